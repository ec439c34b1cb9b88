"""A paged KV cache held in 4 bits: quantise on write, read back, attend.

The cache is one pool of pages for keys and one for values, uint8 tensors
``(num_blocks, block_size/16, 10*head_dim)`` (``kv4_cache`` makes them): 16
tokens of one head take 10*head_dim bytes, 5 bits a value.  Each group of 32
consecutive values of a row holds a bf16 step ``s`` and middle ``m`` and a
4-bit code per value, which reads as ``m + s * (c - 7.5)``:

    s = bf16((max - min) / 15)     (0 where that is below 2^-126)
    m = bf16((max + min) / 2)
    c = round((x - m) / s + 7.5) clamped to 0..15

A group that holds a NaN or an infinity reads as NaN throughout.  The order
of the bytes within a tile is that of the attention kernel's operands (see
csrc/kv4.h); only whole tiles move between pools, pages being copied as bytes.

Page tables, lengths and heads are those of ``paged_decode_attn``: per
(sequence, KV head) a row of page ids ``block_table[b, h]`` and a length.
The operators run on torch's current stream of the tensors' device, allocate
only their outputs and scratch (both through torch, so a call can be captured
in a HIP graph) and never synchronise with the host.  A tensor they write must
not overlap itself (an expanded one) or, but for kv4_append's lengths in place,
one they read.
"""
import ctypes
import functools
import struct

import torch

from . import _lib
from .ops import _u8

# A small call's time is its host time: the operators read each tensor's
# shape, strides and device once and leave to the C ABI what it checks itself.
_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
_I32, _U8, _BF16 = torch.int32, torch.uint8, torch.bfloat16
# arguments of the C calls as blocks of 8-byte words (wgkv_kv4_*_block)
_pack_append = struct.Struct("32q").pack
_pack_read = struct.Struct("23q").pack
_pack_attn = struct.Struct("20qd3q").pack
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


def kv4_cache_shape(num_blocks, block_size, head_dim):
    """Shape of a pool of ``num_blocks`` pages of ``block_size`` tokens."""
    if block_size not in (16, 32, 64):
        raise ValueError("block_size must be 16, 32 or 64")
    if head_dim not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    return num_blocks, block_size // 16, 10 * head_dim


def kv4_cache(num_blocks, block_size, head_dim, device="cuda"):
    """A pair of empty pools (keys, values)."""
    shape = kv4_cache_shape(num_blocks, block_size, head_dim)
    return tuple(torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))


def _host_tensor():
    raise ValueError("wgkv kernels take device tensors (no CPU fallback)")


def _two_devices():
    raise ValueError("all tensors must be on one device")


def _stream(index):
    raw = _lib._raw_stream
    return raw(index) if raw is not None else torch.cuda.current_stream(index).cuda_stream


def _check_cache(k_cache, v_cache):
    shape = k_cache.shape
    if len(shape) != 3 or v_cache.shape != shape or shape[2] not in (640, 1280) or shape[1] not in (1, 2, 4):
        raise AssertionError("k_cache/v_cache must be (num_blocks, block_size/16, 10*head_dim), as kv4_cache makes them")
    if k_cache.dtype is not _U8 or v_cache.dtype is not _U8:
        raise TypeError("k_cache/v_cache must be uint8")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache/v_cache must be contiguous")
    return shape[0], shape[1] * 16, shape[2] // 10


def _check_heads(block_table, lengths, B, H):
    """The page table and the lengths, copied where their last dimension is
    not contiguous, with their strides and the table's width."""
    shape = block_table.shape
    if len(shape) != 3 or shape[0] != B or shape[1] != H:
        raise AssertionError("block_table must be (batch, num_kv_heads, max_blocks)")
    if lengths.shape != (B, H):
        raise AssertionError("lengths must be (batch, num_kv_heads)")
    if block_table.dtype is not _I32 or lengths.dtype is not _I32:
        raise TypeError("block_table and lengths must be int32")
    bs, ls = block_table.stride(), lengths.stride()
    if bs[2] != 1:
        block_table = block_table.contiguous()
        bs = block_table.stride()
    if ls[1] != 1:
        lengths = lengths.contiguous()
        ls = lengths.stride()
    return block_table, bs, shape[2], lengths, ls[0]


def _rows(t, unit, copy=True):
    """t, its address and strides if its rows can be read and written 16
    bytes (``unit`` elements) at a time, else (``copy``) a contiguous copy's,
    or None."""
    st = t.stride()
    p = t.data_ptr()
    if st[3] == 1 and not (st[0] | st[1] | st[2]) % unit and not p % 16:
        return t, p, st
    # the stride of a dimension of one entry means nothing
    sz = tuple(0 if n == 1 else x for n, x in zip(t.shape, st))
    if st[3] == 1 and not (sz[0] | sz[1] | sz[2]) % unit and not p % 16:
        return t, p, sz
    if not copy:
        return None
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), t.stride()


_COUNTS_ITSELF = 16384  # tokens of a mask that the append counts in its own launch


def kv4_append(k, v, k_cache, v_cache, block_table, lengths, g_mask=None, out=None, status=None):
    """Quantise tokens into the heads' pages behind the ones already there.

    k, v (B, T, Hkv, D) bf16, fp16 or fp32 in any layout; the tokens with
    ``g_mask`` (B, Hkv, T) nonzero -- all without it -- go, in order, to
    positions lengths[b, h], lengths[b, h] + 1, ... of their head, whose page
    ``p // block_size`` is ``block_table[b, h, p // block_size]``: pages are
    the caller's to provide, and those written must stand in the table once.
    Tokens the mask leaves out are not read into the cache whatever they hold
    (padding, NaN), and bytes of other tokens are left as they were.

    Returns the new lengths, int32 (B, Hkv): ``out`` where given, which may
    be ``lengths`` itself.  Lengths never exceed max_blocks * block_size: what
    has no room is dropped, as is a token whose page id is outside the pool
    (its position stays used), and then ``status`` (int32, optional) is set
    to WGKV_ERR_CAPACITY, as the dual cache's is.
    """
    num_blocks, P, D = _check_cache(k_cache, v_cache)
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or shape[3] != D:
        raise AssertionError("k/v must be (batch, tokens, num_kv_heads, head_dim)")
    B, T, H, _ = shape
    code = _DTYPES.get(k.dtype)
    if code is None or v.dtype is not k.dtype:
        raise TypeError("k/v must be bf16, fp16 or fp32, both alike")
    if out is not None and (out.shape != (B, H) or out.dtype is not _I32 or (H > 1 and out.stride(1) != 1)):
        raise AssertionError("out must be int32 (batch, num_kv_heads), heads contiguous")
    if status is not None and (status.dtype is not _I32 or status.numel() < 1):
        raise TypeError("status must be an int32 tensor")
    if g_mask is not None and g_mask.shape != (B, H, T):
        raise AssertionError("g_mask must be (batch, num_kv_heads, tokens)")
    table, bs, width, lens, ls = _check_heads(block_table, lengths, B, H)
    dev = k.get_device()
    if dev < 0:
        _host_tensor()
    if (v.get_device() != dev or k_cache.get_device() != dev or v_cache.get_device() != dev or table.get_device() != dev
            or lens.get_device() != dev or (g_mask is not None and g_mask.get_device() != dev)
            or (out is not None and out.get_device() != dev) or (status is not None and status.get_device() != dev)):
        _two_devices()
    if dev != _current_device():  # a null stream is the current device's
        with torch.cuda.device(dev):
            return kv4_append(k, v, k_cache, v_cache, block_table, lengths, g_mask, out, status)
    mp, ms = 0, (0, 0)
    if g_mask is not None:
        m = _u8(g_mask)
        if T > 1 and m.stride(2) != 1:
            m = m.contiguous()
        ms = m.stride()
        mp = m.data_ptr()
    unit = 4 if code == 1 else 8
    k, kp, ks = _rows(k, unit)
    v, vp, vs = _rows(v, unit)
    given = out is not None
    if not given:
        out = torch.empty_like(lens, memory_format=torch.contiguous_format)
    L = _lib.lib()
    # a launch before counts the mask, and copies lengths written in place
    counted = T > 256 and (given or (g_mask is not None and T > _COUNTS_ITSELF))
    nbytes = L.wgkv_kv4_append_workspace_bytes(B, H, T) if counted else 0
    ws = torch.empty(nbytes, dtype=_U8, device=dev) if nbytes else None
    st = L.wgkv_kv4_append_block(_pack_append(
        kp, ks[0], ks[1], ks[2], vp, vs[0], vs[1], vs[2], code, mp, ms[0], ms[1],
        lens.data_ptr(), ls, out.data_ptr(), out.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), num_blocks, P,
        table.data_ptr(), bs[0], bs[1], width, B, T, H, D,
        0 if status is None else status.data_ptr(), 0 if ws is None else ws.data_ptr(), nbytes, _stream(dev)))
    if st:
        _lib.check(st, "wgkv_kv4_append")
    return out


def kv4_read(k_cache, v_cache, block_table, lengths, rows, starts=None, dtype=torch.bfloat16, out=None):
    """The cache's rows as dense tensors: (k, v), each (B, rows, Hkv, D) of
    ``dtype`` (bf16, fp16 or fp32).

    Row i of head (b, h) is position ``starts[b, h] + i`` (``starts`` int32
    (B, Hkv), optional: 0), and zeros from the head's length on and where the
    page id is outside the pool.  ``out`` (optional) is the pair of tensors
    to fill (through a copy where their rows are not 16-byte aligned).
    """
    num_blocks, P, D = _check_cache(k_cache, v_cache)
    B, H = lengths.shape if lengths.dim() == 2 else (-1, -1)
    table, bs, width, lens, ls = _check_heads(block_table, lengths, B, H)
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError("kv4_read gives bf16, fp16 or fp32")
    if rows < 0:
        raise AssertionError("rows must not be negative")
    sp, ss = 0, 0
    if starts is not None:
        if starts.shape != (B, H) or starts.dtype is not _I32:
            raise AssertionError("starts must be int32 (batch, num_kv_heads)")
        if starts.stride(1) != 1:
            starts = starts.contiguous()
        sp, ss = starts.data_ptr(), starts.stride(0)
    dev = k_cache.get_device()
    if dev < 0:
        _host_tensor()
    if (v_cache.get_device() != dev or table.get_device() != dev or lens.get_device() != dev
            or (starts is not None and starts.get_device() != dev)):
        _two_devices()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return kv4_read(k_cache, v_cache, block_table, lengths, rows, starts, dtype, out)
    if out is None:
        ko = torch.empty((B, rows, H, D), dtype=dtype, device=dev)
        vo = torch.empty_like(ko)
        out = (ko, vo)
        st = ko.stride()
        kp, vp = ko.data_ptr(), vo.data_ptr()
    else:
        ko, vo = out
        if ko is vo:
            raise AssertionError("out must be two tensors")
        if ko.shape != (B, rows, H, D) or vo.shape != ko.shape or ko.dtype != dtype or vo.dtype != dtype:
            raise AssertionError("out must be two (batch, rows, num_kv_heads, head_dim) tensors of dtype")
        if ko.get_device() != dev or vo.get_device() != dev:
            _two_devices()
        unit = 4 if code == 1 else 8
        kr, vr = _rows(ko, unit, False), _rows(vo, unit, False)
        if kr is None or vr is None or kr[2] != vr[2]:  # no rows of 16-byte steps, or two layouts
            for dst, src in zip(out, kv4_read(k_cache, v_cache, table, lens, rows, starts, dtype)):
                dst.copy_(src)
            return out
        _, kp, st = kr
        vp = vr[1]
    if rows == 0:
        return out
    err = _lib.lib().wgkv_kv4_read_block(_pack_read(
        k_cache.data_ptr(), v_cache.data_ptr(), num_blocks, P, table.data_ptr(), bs[0], bs[1], width,
        lens.data_ptr(), ls, sp, ss, kp, vp, st[0], st[1], st[2], code, B, rows, H, D, _stream(dev)))
    if err:
        _lib.check(err, "wgkv_kv4_read")
    return out


_COUNTERS = 8192  # bytes at the start of the attention's workspace that must be zero
_KEPT = 32  # streams whose scratch is kept, the last to have asked for one
_workspaces = {}
_captured = {}


@functools.lru_cache(maxsize=None)
def _attn_bytes(Hq, H, D):
    return _lib.lib().wgkv_kv4_decode_workspace_bytes(Hq, H, D)


def _attn_workspace(dev, stream, nbytes):
    """Scratch of the attention, its arrival counters zero.  One per device
    and stream: calls on a stream run in turn and leave the counters zero, and
    calls on two streams never meet.  Captured calls get scratch from their
    graph's memory, cleared by the graph, since two graphs that were captured
    on one stream may run on two: one per capture and stream, for the calls
    that a graph holds of a stream run in turn too (32 calls of 8 heads x 1300
    tokens: 9.6 us each, 10.9 with scratch for each).

    Letting scratch go is safe at any time: its memory then serves later calls
    of the same stream, or stays with the graph.  A capture's is held up to
    the next capture's first call or the next uncaptured one, so that a graph
    that is gone can return its memory; a stream's until _KEPT others had
    theirs, since streams come and go."""
    key = (dev, stream)
    if _capturing():
        capture = ctypes.c_uint64()
        _lib.check(_lib.lib().wgkv_stream_capture_id(stream, ctypes.byref(capture)), "wgkv_stream_capture_id")
        now = capture.value
        held, ws = _captured.get(key, (0, None))
        if not now or held != now or ws.numel() < nbytes:
            ws = torch.empty(nbytes, dtype=_U8, device=dev)
            ws[:_COUNTERS].zero_()
            for other, (i, _) in list(_captured.items()):
                if i != now:
                    _captured.pop(other, None)
            if now:  # 0: a capture that was invalidated
                _captured[key] = (now, ws)
        return ws
    if _captured:
        _captured.clear()
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(nbytes, dtype=_U8, device=dev)
        _workspaces.pop(key, None)
        _workspaces[key] = ws
        for other in list(_workspaces)[:-_KEPT]:
            _workspaces.pop(other, None)
    return ws


def paged_decode_attn_kv4(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, out=None):
    """``paged_decode_attn`` over a 4-bit cache: q (B, 1, Hq, D) bf16 attends
    to the first cache_seqlens[b, h] tokens of its KV head; returns (B, 1, Hq,
    D) bf16, zeros for a head without tokens.  Hq / Hkv may be up to 8, B * Hkv
    up to 2048.  The probabilities, times their value's step, are rounded to
    bf16 for their product with the codes (outputs are 2.1e-3 to 2.4e-3 off, rms
    over rms, of which their own rounding is 1.7e-3); sums are fp32, before their division by the probabilities' sum
    (so values beyond 2^100 may overflow to NaN).  Tokens whose score falls
    below fp32's range weigh nothing, and a head that has no others gives zeros.
    Lengths and page ids out of range are clamped to the table and the pool."""
    num_blocks, P, D = _check_cache(k_cache, v_cache)
    shape = q.shape
    if len(shape) != 4 or shape[1] != 1 or shape[3] != D:
        raise AssertionError("q must be (batch, 1, num_query_heads, head_dim)")
    B, _, Hq, _ = shape
    if q.dtype is not _BF16:
        raise TypeError("q must be bf16")
    H = cache_seqlens.shape[1] if cache_seqlens.dim() == 2 else -1
    table, bs, width, lens, ls = _check_heads(block_table, cache_seqlens, B, H)
    if H < 1 or Hq % H:
        raise AssertionError("num_query_heads must be a multiple of num_kv_heads")
    dev = q.get_device()
    if dev < 0:
        _host_tensor()
    if (k_cache.get_device() != dev or v_cache.get_device() != dev or table.get_device() != dev
            or lens.get_device() != dev or (out is not None and out.get_device() != dev)):
        _two_devices()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return paged_decode_attn_kv4(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, out)
    q, qp, qs = _rows(q, 8)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        op, os = out.data_ptr(), out.stride()
    else:
        if out.shape != shape or out.dtype is not _BF16:
            raise AssertionError("out must be (batch, 1, num_query_heads, head_dim) bf16")
        rows = _rows(out, 8, False)
        if rows is None:  # they cannot be written 16 bytes at a time
            return out.copy_(paged_decode_attn_kv4(q, k_cache, v_cache, lens, table, softmax_scale))
        _, op, os = rows
    L = _lib.lib()
    stream = _stream(dev)
    ws = _attn_workspace(dev, stream, _attn_bytes(Hq, H, D))
    st = L.wgkv_kv4_decode_attn_block(_pack_attn(
        qp, qs[0], qs[2], k_cache.data_ptr(), v_cache.data_ptr(), num_blocks, P, lens.data_ptr(), ls,
        table.data_ptr(), bs[0], bs[1], width, op, os[0], os[2], B, Hq, H, D, softmax_scale, ws.data_ptr(), ws.numel(),
        stream))
    if st:
        _lib.check(st, "wgkv_kv4_decode_attn")
    return out
