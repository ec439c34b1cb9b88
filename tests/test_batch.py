"""The packed-batch serving operators, host only: the oracle against a second
reading of the definitions, and the calls that are refused (argument checks run
before any HIP call)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import batch as ob

I32, BF16 = torch.int32, torch.bfloat16


def test_oracle_tables_by_hand():
    table = np.full((2, 1, 4), -1, dtype=np.int32)
    table[0, 0, 0] = 9
    lens, slots, out, state, status = ob.tables([[15], [0]], [0, 2, 19], 20, table, [4, 2], 16, 16, None, [11, 12, 13])
    assert lens.tolist() == [[17], [17]] and status == 0
    # request 0 fills page 9 and takes the first of the list's last entries; request 1 the next and a fresh one
    assert out[0, 0].tolist() == [9, 11, -1, -1] and out[1, 0].tolist() == [12, 4, -1, -1]
    assert slots[:, 0].tolist() == [9 * 16 + 15, 11 * 16] + [12 * 16 + i for i in range(16)] + [4 * 16, -1]
    assert state.tolist() == [5, 0]


def test_oracle_prompt_by_hand():
    """Values that name their key: the output is the mean of the visible keys' names."""
    n, W, S = 9, 3, 2
    q = torch.zeros(n, 1, 4)
    k = torch.randn(n, 1, 4, generator=torch.Generator().manual_seed(0))
    v = torch.arange(float(n))[:, None, None].expand(n, 1, 4)
    out, _ = ob.prompt(q, k, v, [0, n], [0, n], W, S, 1.0)
    for p in range(n):
        seen = [j for j in range(n) if j <= p and (j > p - W or j < S)]
        assert abs(out[p, 0, 0].item() - sum(seen) / len(seen)) < 1e-12
    out, _ = ob.prompt(q, k[:4], v[:4], [0, n], [0, 4], W, S, 1.0)  # five rows see nothing
    assert not out[:5].any() and out[8, 0, 0].item() == pytest.approx((0 + 1 + 2 + 3) / 4)


def host():
    k = torch.zeros(3, 2, 64, dtype=BF16)
    kc = torch.zeros(8, 16, 64, dtype=BF16)
    return dict(k=k, v=k.clone(), q=torch.zeros(3, 4, 64, dtype=BF16), q1=torch.zeros(2, 1, 4, 64, dtype=BF16), kc=kc,
                vc=kc.clone(), table=torch.zeros(2, 2, 4, dtype=I32), lens=torch.zeros(2, 2, dtype=I32),
                cu=torch.tensor([0, 1, 3], dtype=I32), state=torch.zeros(2, dtype=I32),
                slots=torch.zeros(3, 2, dtype=I32))


def test_tables_refusals():
    import wgkv
    x = host()
    good = (x["lens"], x["cu"], 3, x["table"], x["state"], 8, 16)
    for i, bad, err in [(0, x["lens"][:1], AssertionError), (0, x["lens"].long(), TypeError),
                        (1, x["cu"][:2], AssertionError), (1, x["cu"].long(), TypeError),
                        (1, x["cu"][None], AssertionError), (1, x["cu"][:1], AssertionError),
                        (2, -1, AssertionError),
                        (3, x["table"][0], AssertionError), (3, x["table"].long(), TypeError),
                        (3, torch.zeros(2, 2, 8, dtype=I32)[..., ::2], ValueError),
                        (4, torch.zeros(3, dtype=I32), AssertionError), (4, x["state"].long(), AssertionError),
                        (4, torch.zeros(4, dtype=I32)[::2], AssertionError)]:
        with pytest.raises(err):
            wgkv.build_block_tables(*good[:i], bad, *good[i + 1:])
    for kw, err in [(dict(g_mask=torch.ones(3, 2)), AssertionError), (dict(free_ids=torch.zeros(3)), AssertionError),
                    (dict(free_ids=torch.zeros(6, dtype=I32)[::2]), AssertionError),
                    (dict(out=torch.zeros(2, 2)), AssertionError), (dict(state_out=torch.zeros(3, dtype=I32)), AssertionError),
                    (dict(slots=torch.zeros(2, 3, dtype=I32)), AssertionError),
                    (dict(slots=torch.zeros(3, 4, dtype=I32)[:, ::2]), AssertionError),
                    (dict(status=torch.zeros(1)), TypeError), (dict(), ValueError)]:
        with pytest.raises(err):
            wgkv.build_block_tables(*good, **kw)


def test_append_refusals():
    import wgkv
    x = host()
    good = (x["k"], x["v"], x["kc"], x["vc"], x["slots"])
    for i, bad, err in [(0, x["k"][0], AssertionError), (0, x["k"][:, :1], AssertionError), (0, x["k"].float(), TypeError),
                        (1, x["v"].half(), TypeError), (2, x["kc"][..., :32], AssertionError),
                        (2, x["kc"].float(), TypeError), (2, x["kc"][::2], AssertionError), (4, x["slots"].long(), TypeError),
                        (4, x["slots"].t(), AssertionError), (4, x["slots"], ValueError)]:
        with pytest.raises(err):
            wgkv.paged_append(*good[:i], bad, *good[i + 1:])
    wide = torch.zeros(16, 16, 64, dtype=BF16)
    with pytest.raises(ValueError):
        wgkv.paged_append(x["k"], x["v"], wide[::2], wide[1::2], x["slots"])


def test_prompt_refusals():
    import wgkv
    x = host()
    good = (x["q"], x["k"], x["v"], x["cu"], 4, 1)
    for i, bad, err in [(0, x["q"][None], AssertionError), (0, x["q"][:, :3], AssertionError), (0, x["q"].float(), TypeError),
                        (0, x["q"][..., :32], AssertionError), (1, x["k"][:2], AssertionError), (1, x["k"].half(), TypeError),
                        (3, x["cu"].long(), TypeError), (3, x["cu"][:1], AssertionError), (4, 0, ValueError),
                        (5, -1, ValueError), (5, 1, ValueError)]:
        with pytest.raises(err):
            wgkv.sink_window_attn(*good[:i], bad, *good[i + 1:])
    with pytest.raises(AssertionError):
        wgkv.sink_window_attn(*good, cu_seqlens_k=x["cu"][:2])


def test_token_refusals():
    import wgkv
    x = host()
    win = lambda a, **kw: wgkv.paged_decode_attn_window(*a, 4, 1, 0.1, **kw)  # noqa: E731
    shr = lambda a, **kw: wgkv.paged_decode_attn_shared(*a, x["lens"][:1], x["table"][:1], x["cu"][:2], 0.1, **kw)  # noqa: E731
    good = (x["q1"], x["kc"], x["vc"], x["lens"], x["table"])
    for call in (win, shr):
        for i, bad, err in [(0, x["q1"][:, 0], AssertionError), (0, x["q1"].float(), TypeError),
                            (0, x["q1"][..., :32], AssertionError), (0, x["q1"][:, :, :3], AssertionError),
                            (1, x["kc"].float(), TypeError), (1, x["kc"][::2], AssertionError),
                            (3, x["lens"].long(), TypeError), (3, x["lens"][:1], AssertionError),
                            (4, x["table"].long(), TypeError), (4, x["table"][:, :1], AssertionError),
                            (4, x["table"], ValueError)]:
            with pytest.raises(err):
                call((*good[:i], bad, *good[i + 1:]))
    for w, s in ((0, 1), (4, -1)):
        with pytest.raises(ValueError):
            wgkv.paged_decode_attn_window(*good, w, s, 0.1)
    for i, bad, err in [(0, x["lens"], AssertionError), (1, x["table"], AssertionError), (1, x["table"][:1].long(), TypeError),
                        (2, x["cu"], AssertionError), (2, x["cu"][:2].long(), TypeError), (2, x["cu"][:1], AssertionError)]:
        rest = (x["lens"][:1], x["table"][:1], x["cu"][:2])
        with pytest.raises(err):
            wgkv.paged_decode_attn_shared(*good, *rest[:i], bad, *rest[i + 1:], 0.1)


def test_c_entry_points_check_arguments_without_gpu():
    """Every refusal below is decided before any HIP call."""
    from wgkv import _lib
    L = _lib.lib()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) & ~255
    ARG, UNS, WS = _lib.ERR_ARG, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE

    def refused(fn, good, cases):
        for i, bad, st in cases:
            a = list(good)
            a[i] = bad
            assert fn(*a) == st, (i, bad)

    tables = [p, 2, p, 3, None, 0, p, 8, 4, 4, p, p, None, 0, 8, 16, p, 2, p, 2, 2, None, None, 0, None]
    refused(L.wgkv_build_block_tables, tables, [
        (0, None, ARG), (2, None, ARG), (3, -1, ARG), (6, None, ARG), (9, 0, ARG), (10, None, ARG), (11, None, ARG),
        (13, 5, ARG), (14, 0, ARG), (15, 8, UNS), (15, 128, UNS), (14, 1 << 28, UNS), (9, 1 << 27, UNS), (16, None, ARG),
        (18, None, ARG), (19, 0, ARG), (20, 0, ARG), (20, 1 << 24, UNS),
        (7, 0, ARG), (8, 3, ARG), (17, 0, ARG),      # table rows or lengths that meet
        (3, 300, WS), (3, 0x7fffffff, UNS)])
    assert L.wgkv_block_tables_workspace_bytes(2, 2, 256) == 0 < L.wgkv_block_tables_workspace_bytes(2, 2, 257)
    append = [p, 128, 64, p, 128, 64, p, p + 1024, 8, p, 3, 2, 64, None]
    refused(L.wgkv_paged_append, append, [
        (0, None, ARG), (3, None, ARG), (6, None, ARG), (9, None, ARG), (10, -1, ARG), (11, 0, ARG), (12, 0, ARG),
        (12, 60, UNS), (0, p + 2, UNS), (1, 129, UNS), (8, 1 << 32, UNS), (8, -1, ARG), (7, p + 512, ARG), (7, p, ARG)])
    prompt = [p, 256, 64, p, 128, 64, p, 128, 64, p, 256, 64, p, p, 2, 3, 3, 4, 2, 64, 4, 1, 0.1, 0, None, 0, None]
    refused(L.wgkv_sink_window_attn, prompt, [
        (0, None, ARG), (3, None, ARG), (9, None, ARG), (12, None, ARG), (13, None, ARG), (14, 0, ARG), (14, 2049, UNS),
        (15, -1, ARG), (16, -1, ARG), (17, 3, ARG), (17, 18, UNS), (19, 96, UNS), (20, 0, ARG), (21, -1, ARG),
        (0, p + 2, UNS), (1, 260, UNS), (10, 64, ARG), (10, 0, ARG), (11, 0, ARG), (15, (1 << 30) + 1, UNS)])
    refused(L.wgkv_sink_window_attn, prompt[:14] + [2048] + prompt[15:], [(15, 1 << 26, UNS)])  # rows of all sequences
    few = prompt[:16] + [4000] + prompt[17:20] + [4000] + prompt[21:]  # few rows, many keys: cut into parts
    need = L.wgkv_sink_window_workspace_bytes(2, 3, 4000, 4, 2, 64, 4000, 1)
    assert need > 0 == L.wgkv_sink_window_workspace_bytes(2, 3, 4000, 4, 2, 64, 200, 1)
    refused(L.wgkv_sink_window_attn, few[:24] + [p, need, None], [(24, None, WS), (25, need - 1, WS), (24, p + 4, WS)])
    window = [p, 256, 64, p, p, 8, 16, p, 2, p, 8, 4, 4, p, 256, 64, 2, 4, 2, 64, 4, 1, 0.1, p, 1 << 40, None]
    refused(L.wgkv_paged_decode_attn_window, window, [
        (0, None, ARG), (3, None, ARG), (5, 0, ARG), (6, 8, UNS), (7, None, ARG), (9, None, ARG), (12, 0, ARG),
        (12, 1 << 27, UNS), (13, None, ARG), (14, 0, ARG), (16, 0, ARG), (16, 1025, UNS), (17, 3, ARG), (17, 18, UNS),
        (19, 32, UNS), (20, 0, ARG), (21, -1, ARG), (0, p + 8, UNS), (23, None, WS), (24, 100, WS), (23, p + 4, WS)])
    shared = [p, 256, 64, p, p, 8, 16, p, 2, p, 8, 4, 4, p, 2, p, 8, 4, 4, p, 1, p, 256, 64, 2, 4, 2, 64, 0.1, p, 1 << 40,
              None]
    refused(L.wgkv_shared_decode_attn, shared, [
        (0, None, ARG), (4, None, ARG), (5, 0, ARG), (6, 8, UNS), (7, None, ARG), (12, 0, ARG), (13, None, ARG),
        (15, None, ARG), (18, 0, ARG), (18, 1 << 27, UNS), (19, None, ARG), (20, 0, ARG),
        (20, 1025, UNS), (21, None, ARG), (22, 0, ARG), (24, 0, ARG), (24, 1025, UNS), (25, 3, ARG), (25, 18, UNS),
        (27, 96, UNS), (0, p + 8, UNS), (1, 260, UNS), (29, None, WS), (30, 100, WS)])


def test_block_words_that_do_not_fit():
    from wgkv import _lib, batch
    L = _lib.lib()
    assert L.wgkv_build_block_tables_block(batch._pack_tables(*([1] * 3), 1 << 40, *([1] * 21))) == _lib.ERR_UNSUPPORTED
    assert L.wgkv_paged_append_block(batch._pack_append(*([1] * 10), 1 << 40, 1, 1, 1)) == _lib.ERR_UNSUPPORTED
    assert L.wgkv_sink_window_attn_block(batch._pack_prompt(*([1] * 14), 1 << 40, *([1] * 7), 1.0, 1, 1, 1, 1)) == \
        _lib.ERR_UNSUPPORTED
    assert L.wgkv_paged_decode_attn_window_block(batch._pack_window(*([1] * 6), 1 << 40, *([1] * 15), 1.0, 1, 1, 1)) == \
        _lib.ERR_UNSUPPORTED
    assert L.wgkv_shared_decode_attn_block(batch._pack_shared(*([1] * 6), 1 << 40, *([1] * 21), 1.0, 1, 1, 1)) == \
        _lib.ERR_UNSUPPORTED


def test_meta_shapes():
    import wgkv  # noqa: F401
    m = dict(device="meta")
    q = torch.empty(9, 8, 64, dtype=BF16, **m).transpose(0, 1)
    k, cu = torch.empty(8, 2, 64, dtype=BF16, **m), torch.empty(3, dtype=I32, **m)
    out = torch.ops.wgkv.sink_window_attn(q, k, k, cu, 5, 1)
    assert out.shape == q.shape and out.dtype == BF16 and out.is_contiguous()
    q = torch.empty(2, 1, 8, 64, dtype=BF16, **m)
    kc, ln, tb = torch.empty(9, 16, 64, dtype=BF16, **m), torch.empty(2, 2, dtype=I32, **m), torch.empty(2, 2, 4, dtype=I32, **m)
    assert torch.ops.wgkv.paged_decode_attn_window(q, kc, kc, ln, tb, 5, 1, 0.1).shape == q.shape
    assert torch.ops.wgkv.paged_decode_attn_shared(q, kc, kc, ln, tb, ln[:1], tb[:1], cu[:2], 0.1).shape == q.shape
