"""The 4-bit cache, host only: the oracle's format against its definition,
and the calls that are refused (argument checks run before any HIP call)."""
import numpy as np
import pytest
import torch

from oracle import kv4 as ok


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys", [True, False])
def test_oracle_tile_round_trip(D, keys):
    """Every code, step and middle has its own place in a tile."""
    rng = np.random.default_rng(D + keys)
    places = set()
    for t in range(16):
        for d in range(D):
            at, sh = ok.offsets(t, d, D, keys)
            places.add((int(at), int(sh)))
    assert places == {(a, s) for a in range(8 * D) for s in (0, 4)}
    tile = np.full(10 * D, 0xA5, np.uint8)
    c = rng.integers(0, 16, (16, D))
    s, m = ok.bf16(rng.uniform(0, 2, (16, D // 32))), ok.bf16(rng.normal(size=(16, D // 32)))
    for t in rng.permutation(16):
        ok.put(tile, t, c[t], s[t], m[t], keys)
    for t in range(16):
        for got, want in zip(ok.get(tile, t, D, keys), (c[t], s[t], m[t])):
            assert np.array_equal(got, want)


@pytest.mark.parametrize("mean", [0.0, 3.0, 1e4])
def test_oracle_quantisation_error(mean):
    """|value - x| <= s/2 and what the rounded m and s cost: half a bf16 step
    (2^-8 relative) of m, and 7.5 s 2^-8 at the ends of the range."""
    x = np.random.default_rng(1).normal(size=(200, 64)) + mean
    c, s, m = ok.quantise(x)
    sw, mw = np.repeat(s, 32, 1), np.repeat(m, 32, 1)
    assert (np.abs(ok.values(c, s, m) - x) <= sw / 2 + np.abs(mw) * 2.0 ** -8 + 7.5 * sw * 2.0 ** -8 + 1e-12).all()


def test_oracle_special_groups():
    x = np.zeros((5, 64))
    x[0, :32] = -2.5          # constant: reads exactly
    x[1, 3] = np.inf
    x[2, 40] = np.nan
    x[3, :32] = np.linspace(-3e38, 3e38, 32)
    x[4, :32] = np.linspace(0, 1e-40, 32)  # a step below 2^-126 is 0
    v = ok.values(*ok.quantise(x))
    assert (v[0, :32] == -2.5).all() and (v[0, 32:] == 0).all()
    assert np.isnan(v[1, :32]).all() and (v[1, 32:] == 0).all()
    assert (v[2, :32] == 0).all() and np.isnan(v[2, 32:]).all()
    assert np.isfinite(v[3]).all() and np.abs(v[3, :32] - x[3, :32]).max() <= 6e38 / 30 * 1.02
    assert (np.abs(v[4] - x[4]) <= 1e-40).all()


def _args(B=2, T=3, H=2, D=64, P=16, blocks=4):
    k = torch.zeros(B, T, H, D, dtype=torch.bfloat16)
    kc = torch.zeros(8, P // 16, 10 * D, dtype=torch.uint8)
    return (k, k.clone(), kc, kc.clone(), torch.zeros(B, H, blocks, dtype=torch.int32),
            torch.zeros(B, H, dtype=torch.int32))


def test_append_refusals():
    import wgkv
    k, v, kc, vc, bt, sl = _args()
    for bad, err in [
        ((k[0], v, kc, vc, bt, sl), AssertionError),
        ((k, v[:, :2], kc, vc, bt, sl), AssertionError),
        ((k.double(), v.double(), kc, vc, bt, sl), TypeError),
        ((k, v.float(), kc, vc, bt, sl), TypeError),
        ((k[..., :32], v[..., :32], kc, vc, bt, sl), AssertionError),
        ((k, v, kc.int(), vc, bt, sl), TypeError),
        ((k, v, kc, vc[:4], bt, sl), AssertionError),
        ((k, v, kc[..., :320], vc[..., :320], bt, sl), AssertionError),
        ((k, v, torch.cat([kc, kc])[::2], torch.cat([vc, vc])[::2], bt, sl), ValueError),
        ((k, v, kc, vc, bt[:1], sl), AssertionError),
        ((k, v, kc, vc, bt.long(), sl), TypeError),
        ((k, v, kc, vc, bt, sl[:, :1]), AssertionError),
        ((k, v, kc, vc, bt, sl.long()), TypeError),
        ((k, v, kc, vc, bt, sl), ValueError),  # host tensors
    ]:
        with pytest.raises(err):
            wgkv.kv4_append(*bad)
    for kw, err in [(dict(g_mask=torch.ones(2, 3, 2)), AssertionError),
                    (dict(out=torch.zeros(2, 2)), AssertionError),
                    (dict(out=torch.zeros(2, 3, dtype=torch.int32)), AssertionError),
                    (dict(status=torch.zeros(1)), TypeError)]:
        with pytest.raises(err):
            wgkv.kv4_append(k, v, kc, vc, bt, sl, **kw)


def test_read_and_attention_refusals():
    import wgkv
    _, _, kc, vc, bt, sl = _args()
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16)
    for bad, kw, err in [
        ((kc, vc, bt, sl[0], 4), {}, AssertionError),
        ((kc, vc, bt, sl, -1), {}, AssertionError),
        ((kc, vc, bt, sl, 4), dict(dtype=torch.float64), TypeError),
        ((kc, vc, bt, sl, 4), dict(starts=sl.long()), AssertionError),
        ((kc, vc, bt, sl, 4), {}, ValueError),
    ]:
        with pytest.raises(err):
            wgkv.kv4_read(*bad, **kw)
    for bad, kw, err in [
        ((q[:, 0], kc, vc, sl, bt), {}, AssertionError),
        ((torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16), kc, vc, sl, bt), {}, AssertionError),
        ((q.float(), kc, vc, sl, bt), {}, TypeError),
        ((q[:, :, :3], kc, vc, sl, bt), {}, AssertionError),
        ((q, kc, vc, sl.long(), bt), {}, TypeError),
        ((q, kc, vc, sl, bt), {}, ValueError),
    ]:
        with pytest.raises(err):
            wgkv.paged_decode_attn_kv4(*bad, 0.125, **kw)
    for args in [(4, 24, 64), (4, 16, 96)]:
        with pytest.raises(ValueError):
            wgkv.kv4_cache(*args, device="cpu")


def test_c_entry_points_check_arguments_without_gpu():
    from wgkv import _lib
    L = _lib.lib()
    x = 4096  # an aligned, never dereferenced address
    assert L.wgkv_kv4_append_workspace_bytes(1, 8, 256) == 0
    assert L.wgkv_kv4_append_workspace_bytes(2, 3, 257) == 4 * 6 * (1 + 1 + 2)

    def append(key=x, sk=64, dtype=0, cache=x, pages=4, page=16, maxp=4, B=1, T=4, H=1, D=64, ws=None, n=0):
        return L.wgkv_kv4_append(key, sk, sk, sk, x, sk, sk, sk, dtype, None, 0, 0, x, 1, x, 1, cache, x, pages, page,
                                 x, 4, 4, maxp, B, T, H, D, None, ws, n, None)

    for kw, want in [(dict(key=None), _lib.ERR_ARG), (dict(T=-1), _lib.ERR_ARG), (dict(B=0), _lib.ERR_ARG),
                     (dict(maxp=0), _lib.ERR_ARG), (dict(pages=0), _lib.ERR_ARG),
                     (dict(key=x + 2), _lib.ERR_UNSUPPORTED), (dict(sk=60), _lib.ERR_UNSUPPORTED),
                     (dict(dtype=3), _lib.ERR_UNSUPPORTED), (dict(D=96), _lib.ERR_UNSUPPORTED),
                     (dict(page=8), _lib.ERR_UNSUPPORTED), (dict(cache=x + 8), _lib.ERR_UNSUPPORTED),
                     (dict(maxp=1 << 28), _lib.ERR_UNSUPPORTED), (dict(B=256, H=257), _lib.ERR_UNSUPPORTED),
                     (dict(T=257), _lib.ERR_WORKSPACE), (dict(T=257, ws=x, n=8), _lib.ERR_WORKSPACE)]:
        assert append(**kw) == want, kw

    def read(out=x, so=64, rows=4, dtype=0, D=64):
        return L.wgkv_kv4_read(x, x, 4, 16, x, 4, 4, 4, x, 1, None, 0, out, x, so, so, so, dtype, 1, rows, 1, D, None)

    for kw, want in [(dict(out=None), _lib.ERR_ARG), (dict(rows=0), _lib.ERR_ARG), (dict(so=4), _lib.ERR_UNSUPPORTED),
                     (dict(dtype=-1), _lib.ERR_UNSUPPORTED), (dict(D=32), _lib.ERR_UNSUPPORTED)]:
        assert read(**kw) == want, kw


@pytest.mark.parametrize("D,P", [(64, 16), (128, 64)])
def test_dispatcher_operators(D, P):
    """Registered with their schemas; the Meta kernels give the shapes."""
    import wgkv  # noqa: F401
    for n in ("paged_decode_attn_kv4", "kv4_read"):
        assert str(getattr(torch.ops.wgkv, n).default._schema).startswith(f"wgkv::{n}(")
    meta = dict(device="meta")
    kc = torch.empty(7, P // 16, 10 * D, dtype=torch.uint8, **meta)
    q = torch.empty(2, 1, 8, D, dtype=torch.bfloat16, **meta)
    sl, bt = torch.empty(2, 4, dtype=torch.int32, **meta), torch.empty(2, 4, 9, dtype=torch.int32, **meta)
    out = torch.ops.wgkv.paged_decode_attn_kv4(q, kc, kc, sl, bt, 0.1)
    assert out.shape == q.shape and out.dtype == q.dtype
    k, v = torch.ops.wgkv.kv4_read(kc, kc, bt, sl, 33, dtype=torch.float32)
    assert k.shape == v.shape == (2, 33, 4, D) and k.dtype == torch.float32


def test_argument_blocks_are_the_calls_arguments():
    """The block entry points check what the plain ones check (a null query,
    cache or output is refused before any HIP call)."""
    from wgkv import _lib, kv4
    L = _lib.lib()
    assert L.wgkv_kv4_append_block(kv4._pack_append(*[0] * 32)) == _lib.ERR_ARG
    assert L.wgkv_kv4_read_block(kv4._pack_read(*[0] * 23)) == _lib.ERR_ARG
    assert L.wgkv_kv4_decode_attn_block(kv4._pack_attn(*[0] * 20, 1.0, 0, 0, 0)) == _lib.ERR_ARG
    x = 4096
    sizes = dict(append=(len(_lib.SIGNATURES["wgkv_kv4_append"][1]), 32), read=(len(_lib.SIGNATURES["wgkv_kv4_read"][1]), 23),
                 attn=(len(_lib.SIGNATURES["wgkv_kv4_decode_attn"][1]), 24))
    assert all(a == b for a, b in sizes.values()), sizes
    # every word reaches its argument: the last checks before a launch
    words = [x, 64, 64, 64, x, 64, 64, 64, 0, 0, 0, 0, x, 1, x, 1, x, x, 4, 16, x, 4, 4, 4, 1, 257, 1, 64, 0, x, 8, 0]
    assert L.wgkv_kv4_append_block(kv4._pack_append(*words)) == _lib.ERR_WORKSPACE
    words = [x, x, 4, 16, x, 4, 4, 4, x, 1, 0, 0, x, x, 64, 64, 4, 0, 1, 4, 1, 64, 0]
    assert L.wgkv_kv4_read_block(kv4._pack_read(*words)) == _lib.ERR_UNSUPPORTED
    words = [x, 64, 64, x, x, 4, 16, x, 1, x, 4, 4, 4, x, 64, 64, 1, 4, 1, 64, 0.125, x, 8, 0]
    assert L.wgkv_kv4_decode_attn_block(kv4._pack_attn(*words)) == _lib.ERR_WORKSPACE


def test_outputs_that_overlap_are_refused():
    """Lengths written in place or apart from those read, rows written once;
    what passes these checks fails on the missing workspace."""
    import wgkv
    from wgkv import _lib
    L = _lib.lib()
    x = 1 << 20

    def append(new, new_sb, B=3, H=4, len_sb=4):
        return L.wgkv_kv4_append(x, 64, 64, 64, x, 64, 64, 64, 0, x, 0, 0, x, len_sb, new, new_sb, x, x, 4, 16,
                                 x, 4, 4, 4, B, 16385, H, 64, None, None, 0, None)
    for good in [dict(new=x, new_sb=4), dict(new=x + 48, new_sb=4), dict(new=x - 48, new_sb=4),
                 dict(new=x, new_sb=9, B=1),
                 dict(new=x + 16, new_sb=8, len_sb=8), dict(new=x - 16, new_sb=8, len_sb=8),  # slices of one array
                 dict(new=x + 48, new_sb=8, len_sb=8), dict(new=x + 48, new_sb=4, len_sb=0)]:
        assert append(**good) == _lib.ERR_WORKSPACE, good
    for bad in [dict(new=x + 4, new_sb=4), dict(new=x - 44, new_sb=4), dict(new=x + 44, new_sb=4),
                dict(new=x, new_sb=8), dict(new=x + 12, new_sb=8, len_sb=8), dict(new=x - 12, new_sb=8, len_sb=8),
                dict(new=x + 64, new_sb=0), dict(new=x + 4, new_sb=4, B=1), dict(new=x + 64, new_sb=3),
                dict(new=x + 8, new_sb=4, len_sb=0)]:
        assert append(**bad) == _lib.ERR_ARG, bad

    def read(sb=4096, st=128, sh=64, key=x, value=2 * x, B=2, H=2):
        return L.wgkv_kv4_read(x, x, 4, 16, x, 4, 4, 4, x, 2, None, 0, key, value, sb, st, sh, 0, B, 8, H, 64, None)
    for bad in [dict(sb=0), dict(st=0), dict(sh=0), dict(value=x)]:
        assert read(**bad) == _lib.ERR_ARG, bad

    def attend(sb, sh, B=2, Hq=4):
        return L.wgkv_kv4_decode_attn(x, 256, 64, x, x, 4, 16, x, 4, x, 4, 4, 4, 2 * x, sb, sh, B, Hq, 1, 64, 0.1,
                                      None, 0, None)
    assert attend(256, 64) == attend(0, 64, B=1) == attend(64, 0, Hq=1) == _lib.ERR_WORKSPACE
    assert attend(0, 64) == attend(256, 0) == _lib.ERR_ARG
    _, _, kc, vc, bt, sl = _args()
    out = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises((AssertionError, ValueError)):
        wgkv.kv4_read(kc, vc, bt, sl, 4, out=(out, out))


def test_capture_id_needs_somewhere_to_go():
    from wgkv import _lib
    assert _lib.lib().wgkv_stream_capture_id(None, None) == _lib.ERR_ARG


def test_append_refuses_pools_that_meet():
    """Keys and values of one page are written by different lanes: two pools
    that share bytes, wholly or in part, would be left to a race."""
    from wgkv import _lib
    L = _lib.lib()
    x, pages, P, D = 1 << 20, 4, 32, 64
    size = pages * P // 16 * 10 * D

    def append(kc, vc):
        return L.wgkv_kv4_append(x, 64, 64, 64, x, 64, 64, 64, 0, None, 0, 0, x, 1, x, 1, kc, vc, pages, P,
                                 x, 4, 4, 4, 1, 4, 1, D, None, None, 0, None)
    for kc, vc in [(x, x), (x, x + size - 16), (x + size - 16, x), (x, x + 16)]:
        assert append(kc, vc) == _lib.ERR_ARG, (kc, vc)


def test_output_rows_that_meet_are_refused():
    """Rows of an output may lie anyhow but on each other: in strides smaller
    than a row, interleaved, keys' rows among values'."""
    from wgkv import _lib
    L = _lib.lib()
    x = 1 << 20

    def read(sb=4096, st=128, sh=64, apart=1 << 20, B=2, H=2):
        return L.wgkv_kv4_read(x, x, 4, 16, x, 4, 4, 4, x, 2, None, 0, x, x + 2 * apart, sb, st, sh, 0, B, 8, H, 64, None)
    for bad in [dict(st=120), dict(sh=8), dict(sb=8 * 128 - 64), dict(apart=0), dict(apart=56), dict(apart=-56),
                dict(apart=64), dict(apart=4096), dict(apart=8 * 128 - 8), dict(sb=256, st=128, sh=64),
                dict(st=-128, sb=128), dict(sb=1 << 60, st=1 << 61, sh=32)]:
        assert read(**bad) == _lib.ERR_ARG, bad

    def attend(sb, sh, B, Hq):
        return L.wgkv_kv4_decode_attn(x, 256, 64, x, x, 4, 16, x, 4, x, 4, 4, 4, 2 * x, sb, sh, B, Hq, 1, 64, 0.1,
                                      None, 0, None)
    rng = np.random.default_rng(3)
    seen = set()
    for _ in range(2000):
        B, Hq = int(rng.integers(1, 9)), int(rng.integers(1, 9))
        sb, sh = (int(rng.integers(0, 9) * rng.choice([8, 64, 128, 192])) for _ in range(2))
        at = np.sort([b * sb + h * sh for b in range(B) for h in range(Hq)])
        meets = bool((np.diff(at) < 64).any())
        nested = all(s >= 64 and (n == 1 or s >= (n - 1) * t + 64) for s, t, n in [sorted([(sb, sh, Hq), (sh, sb, B)])[1]])
        seen.add((meets, nested))
        assert attend(sb, sh, B, Hq) == (_lib.ERR_ARG if meets else _lib.ERR_WORKSPACE), (B, Hq, sb, sh)
    assert seen >= {(True, False), (False, False), (False, True)}


def test_sizes_past_32_bits_are_refused():
    """The C calls' 32-bit sizes come from 64-bit ones in the argument blocks:
    what does not fit is refused, not cut off (an expanded tensor may have 2^32
    + 1 tokens).  What passes fails on a missing workspace or argument."""
    from wgkv import _lib, kv4
    L = _lib.lib()
    x = 4096
    append = [x, 64, 64, 64, x, 64, 64, 64, 0, 0, 0, 0, x, 1, x, 1, x, x, 4, 16, x, 4, 4, 4, 1, 257, 1, 64, 0, x, 8, 0]
    read = [x, x, 4, 16, x, 4, 4, 4, x, 1, 0, 0, 0, x, 64, 64, 64, 0, 1, 4, 1, 64, 0]
    attn = [x, 64, 64, x, x, 4, 16, x, 1, x, 4, 4, 4, x, 64, 64, 1, 4, 1, 64, 0.125, x, 8, 0]
    for call, pack, words, narrow, otherwise in [
            (L.wgkv_kv4_append_block, kv4._pack_append, append, (8, 19, 23, 24, 25, 26, 27), _lib.ERR_WORKSPACE),
            (L.wgkv_kv4_read_block, kv4._pack_read, read, (3, 7, 17, 18, 19, 20, 21), _lib.ERR_ARG),
            (L.wgkv_kv4_decode_attn_block, kv4._pack_attn, attn, (6, 12, 16, 17, 18, 19), _lib.ERR_WORKSPACE)]:
        assert call(pack(*words)) == otherwise
        for i in narrow:
            for more in (1 << 32, -(1 << 32), 1 << 40):
                wide = list(words)
                wide[i] += more
                assert call(pack(*wide)) == _lib.ERR_UNSUPPORTED, (i, more)


class _Captures:
    """The scratch's view of a capture: its state and id."""

    def __init__(self, monkeypatch):
        from wgkv import kv4
        self.id = 0
        monkeypatch.setattr(kv4, "_capturing", lambda: self.id is not None)
        monkeypatch.setattr(kv4, "_workspaces", {})
        monkeypatch.setattr(kv4, "_captured", {})
        monkeypatch.setattr(kv4._lib, "lib", lambda: self)

    def wgkv_stream_capture_id(self, stream, ref):
        ref._obj.value = self.id
        return 0


def test_scratch_is_let_go(monkeypatch):
    """Attention scratch: a capture's is held no longer than to the next
    capture or uncaptured call, a stream's until many others had theirs."""
    import gc
    import weakref
    from wgkv import kv4
    cap = _Captures(monkeypatch)

    def scratch(stream, n=kv4._COUNTERS + 64):
        return weakref.ref(kv4._attn_workspace("cpu", stream, n))
    cap.id = 7
    a, b = scratch(1), scratch(2)
    assert a() is not None and scratch(1)() is a() and scratch(2)() is b()  # shared within the capture
    big = scratch(1, kv4._COUNTERS + 4096)
    gc.collect()
    assert a() is None and big() is not None and scratch(1)() is big()
    cap.id = 8
    c = scratch(3)
    gc.collect()
    assert big() is None and b() is None and c() is not None  # another capture's
    cap.id = None
    e = scratch(1)
    gc.collect()
    assert c() is None and not kv4._captured
    assert e() is not None and scratch(1)() is e()
    for s in range(100, 400):
        assert int(kv4._attn_workspace("cpu", s, kv4._COUNTERS)[:kv4._COUNTERS].max()) == 0
    gc.collect()
    assert e() is None and len(kv4._workspaces) <= 32
    assert scratch(399)() is not None and int(scratch(1)().max()) == 0


def test_scratch_of_a_capture_without_id(monkeypatch):
    """A capture that was invalidated has no id: scratch of its own, shared
    with no other call."""
    from wgkv import kv4
    cap = _Captures(monkeypatch)
    cap.id = 0
    x, y = (kv4._attn_workspace("cpu", 5, kv4._COUNTERS + 64) for _ in range(2))
    assert x.data_ptr() != y.data_ptr() and not x[:kv4._COUNTERS].any()
