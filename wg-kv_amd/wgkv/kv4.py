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
in a HIP graph) and never synchronise with the host.
"""
import functools

import torch

from . import _lib
from .ops import _u8

_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}


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


def _same_device(first, *rest):
    if not first.is_cuda:
        raise ValueError("wgkv kernels take device tensors (no CPU fallback)")
    dev = first.device
    for t in rest:
        if t is not None and t.device != dev:
            raise ValueError("all tensors must be on one device")
    return dev


def _on_own_device(op):
    """Runs op with its tensors' device current: a null stream, and whether
    a stream is being captured, are the current device's."""
    @functools.wraps(op)
    def call(first, *args, **kw):
        dev = first.device
        if dev.type != "cuda" or dev.index == torch.cuda.current_device():
            return op(first, *args, **kw)
        with torch.cuda.device(dev):
            return op(first, *args, **kw)
    return call


def _call(dev, where, fn, *args):
    st = fn(*args, _lib.stream_handle(dev))
    if st:
        _lib.check(st, where)


def _check_cache(k_cache, v_cache):
    shape = k_cache.shape
    if len(shape) != 3 or v_cache.shape != shape or shape[2] not in (640, 1280) or shape[1] not in (1, 2, 4):
        raise AssertionError("k_cache/v_cache must be (num_blocks, block_size/16, 10*head_dim), as kv4_cache makes them")
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
        raise TypeError("k_cache/v_cache must be uint8")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache/v_cache must be contiguous")
    return shape[0], shape[1] * 16, shape[2] // 10


def _check_heads(block_table, lengths, B, H):
    if block_table.dim() != 3 or block_table.shape[0] != B or block_table.shape[1] != H:
        raise AssertionError("block_table must be (batch, num_kv_heads, max_blocks)")
    if lengths.shape != (B, H):
        raise AssertionError("lengths must be (batch, num_kv_heads)")
    if block_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError("block_table and lengths must be int32")
    if block_table.stride(2) != 1:
        block_table = block_table.contiguous()
    if lengths.stride(1) != 1:
        lengths = lengths.contiguous()
    return block_table, lengths


def _strides(t):
    """Element strides, 0 for dimensions of one entry (theirs mean nothing)."""
    return [0 if n == 1 else s for n, s in zip(t.shape, t.stride())]


def _aligned(t):
    """Whether t's rows can be read and written 16 bytes at a time."""
    unit = 16 // t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and not any(s % unit for s in _strides(t)[:-1])


def _rows(t):
    """t itself where its rows are 16-byte aligned, else a copy."""
    return t if _aligned(t) else t.clone(memory_format=torch.contiguous_format)


@_on_own_device
def kv4_append(k, v, k_cache, v_cache, block_table, lengths, g_mask=None, out=None, status=None):
    """Quantise tokens into the heads' pages behind the ones already there.

    k, v (B, T, Hkv, D) bf16, fp16 or fp32 in any layout; the tokens with
    ``g_mask`` (B, Hkv, T) nonzero -- all without it -- go, in order, to
    positions lengths[b, h], lengths[b, h] + 1, ... of their head, whose page
    ``p // block_size`` is ``block_table[b, h, p // block_size]``: pages are
    the caller's to provide and must not be shared between heads.  Tokens the
    mask leaves out are not read into the cache whatever they hold (padding,
    NaN), and bytes of other tokens are left as they were.

    Returns the new lengths, int32 (B, Hkv): ``out`` where given, which may
    be ``lengths`` itself.  Lengths never exceed max_blocks * block_size: what
    has no room is dropped, as is a token whose page id is outside the pool
    (its position stays used), and then ``status`` (int32, optional) is set
    to WGKV_ERR_CAPACITY, as the dual cache's is.
    """
    num_blocks, P, D = _check_cache(k_cache, v_cache)
    if k.dim() != 4 or v.shape != k.shape or k.shape[3] != D:
        raise AssertionError("k/v must be (batch, tokens, num_kv_heads, head_dim)")
    B, T, H, _ = k.shape
    if k.dtype not in _DTYPES or v.dtype != k.dtype:
        raise TypeError("k/v must be bf16, fp16 or fp32, both alike")
    if out is not None and (out.shape != (B, H) or out.dtype != torch.int32 or (H > 1 and out.stride(1) != 1)):
        raise AssertionError("out must be int32 (batch, num_kv_heads), heads contiguous")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise TypeError("status must be an int32 tensor")
    if g_mask is not None and g_mask.shape != (B, H, T):
        raise AssertionError("g_mask must be (batch, num_kv_heads, tokens)")
    table, lens = _check_heads(block_table, lengths, B, H)
    dev = _same_device(k, v, k_cache, v_cache, table, lens, g_mask, out, status)
    m, ms = None, (0, 0)
    if g_mask is not None:
        m = _u8(g_mask)
        if T > 1 and m.stride(2) != 1:
            m = m.contiguous()
        ms = m.stride()
    k, v = _rows(k), _rows(v)
    ks, vs = _strides(k), _strides(v)
    if out is None:
        out = torch.empty(B, H, dtype=torch.int32, device=dev)
    L = _lib.lib()
    nbytes = L.wgkv_kv4_append_workspace_bytes(B, H, T)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _call(dev, "wgkv_kv4_append", L.wgkv_kv4_append,
          k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], _DTYPES[k.dtype],
          m.data_ptr() if m is not None else None, ms[0], ms[1],
          lens.data_ptr(), lens.stride(0), out.data_ptr(), out.stride(0),
          k_cache.data_ptr(), v_cache.data_ptr(), num_blocks, P,
          table.data_ptr(), table.stride(0), table.stride(1), table.shape[2],
          B, T, H, D,
          status.data_ptr() if status is not None else None,
          ws.data_ptr() if ws is not None else None, nbytes)
    return out


@_on_own_device
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
    table, lens = _check_heads(block_table, lengths, B, H)
    if dtype not in _DTYPES:
        raise TypeError("kv4_read gives bf16, fp16 or fp32")
    if rows < 0:
        raise AssertionError("rows must not be negative")
    if starts is not None:
        if starts.shape != (B, H) or starts.dtype != torch.int32:
            raise AssertionError("starts must be int32 (batch, num_kv_heads)")
        if starts.stride(1) != 1:
            starts = starts.contiguous()
    dev = _same_device(k_cache, v_cache, table, lens, starts)
    if out is None:
        out = tuple(torch.empty(B, rows, H, D, dtype=dtype, device=dev) for _ in range(2))
    ko, vo = out
    if ko.shape != (B, rows, H, D) or vo.shape != ko.shape or ko.dtype != dtype or vo.dtype != dtype:
        raise AssertionError("out must be two (batch, rows, num_kv_heads, head_dim) tensors of dtype")
    _same_device(k_cache, ko, vo)
    if rows == 0:
        return out
    st = _strides(ko)
    if _strides(vo) != st or not (_aligned(ko) and _aligned(vo)):  # rows cannot be written 16 bytes at a time
        for dst, src in zip(out, kv4_read(k_cache, v_cache, table, lens, rows, starts, dtype)):
            dst.copy_(src)
        return out
    _call(dev, "wgkv_kv4_read", _lib.lib().wgkv_kv4_read,
          k_cache.data_ptr(), v_cache.data_ptr(), num_blocks, P,
          table.data_ptr(), table.stride(0), table.stride(1), table.shape[2],
          lens.data_ptr(), lens.stride(0), starts.data_ptr() if starts is not None else None,
          starts.stride(0) if starts is not None else 0,
          ko.data_ptr(), vo.data_ptr(), st[0], st[1], st[2], _DTYPES[dtype],
          B, rows, H, D)
    return out


_COUNTERS = 8192  # bytes at the start of the attention's workspace that must be zero
_workspaces = {}


def _attn_workspace(dev, nbytes):
    """Scratch of the attention, its arrival counters zero.  One per device
    and stream: calls on a stream run in turn and leave the counters zero, and
    calls on two streams never meet.  A captured call gets scratch of its own
    from the graph's memory, cleared by the graph, since two graphs that were
    captured on one stream may run on two."""
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        ws[:_COUNTERS].zero_()
        return ws
    key = (dev.index, _lib.stream_handle(dev))
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
        _workspaces[key] = ws
    return ws


@_on_own_device
def paged_decode_attn_kv4(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, out=None):
    """``paged_decode_attn`` over a 4-bit cache: q (B, 1, Hq, D) bf16 attends
    to the first cache_seqlens[b, h] tokens of its KV head; returns (B, 1, Hq,
    D) bf16, zeros for a head without tokens.  The probabilities are rounded
    to bf16 for their product with the values; sums are fp32.  Lengths and
    page ids out of range are clamped to the table and the pool."""
    num_blocks, P, D = _check_cache(k_cache, v_cache)
    if q.dim() != 4 or q.shape[1] != 1 or q.shape[3] != D:
        raise AssertionError("q must be (batch, 1, num_query_heads, head_dim)")
    B, _, Hq, _ = q.shape
    if q.dtype != torch.bfloat16:
        raise TypeError("q must be bf16")
    H = cache_seqlens.shape[1] if cache_seqlens.dim() == 2 else -1
    table, lens = _check_heads(block_table, cache_seqlens, B, H)
    if H < 1 or Hq % H:
        raise AssertionError("num_query_heads must be a multiple of num_kv_heads")
    dev = _same_device(q, k_cache, v_cache, table, lens, out)
    if out is None:
        out = torch.empty(B, 1, Hq, D, dtype=torch.bfloat16, device=dev)
    elif out.shape != (B, 1, Hq, D) or out.dtype != torch.bfloat16:
        raise AssertionError("out must be (batch, 1, num_query_heads, head_dim) bf16")
    elif not _aligned(out):  # rows cannot be written 16 bytes at a time
        return out.copy_(paged_decode_attn_kv4(q, k_cache, v_cache, lens, table, softmax_scale))
    q = _rows(q)
    qs, os = _strides(q), _strides(out)
    L = _lib.lib()
    ws = _attn_workspace(dev, L.wgkv_kv4_decode_workspace_bytes(Hq, H, D))
    _call(dev, "wgkv_kv4_decode_attn", L.wgkv_kv4_decode_attn,
          q.data_ptr(), qs[0], qs[2], k_cache.data_ptr(), v_cache.data_ptr(), num_blocks, P,
          lens.data_ptr(), lens.stride(0), table.data_ptr(), table.stride(0), table.stride(1), table.shape[2],
          out.data_ptr(), os[0], os[2], B, Hq, H, D, float(softmax_scale), ws.data_ptr(), ws.numel())
    return out
