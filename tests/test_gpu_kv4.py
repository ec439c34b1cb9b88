"""The 4-bit cache's operators against the 64-bit oracle: appended bytes and
read-back values bit for bit, attention within the bound that its roundings
give (oracle.kv4.attend)."""
import numpy as np
import pytest
import torch

from oracle import kv4 as ok

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
I32 = torch.int32


def table_for(tokens, P, gen, spare=0, extra=3):
    """Page ids of heads with these token counts: a permutation of the pool
    (``extra`` pages unused), -1 past the end; (B, H, width + spare)."""
    B, H = tokens.shape
    pages = (tokens + P - 1) // P
    total, width = int(pages.sum()) + extra, max(1, int(pages.max())) + spare
    perm = torch.randperm(total, generator=gen).to(I32)
    bt = torch.full((B, H, width), -1, dtype=I32)
    off = 0
    for b in range(B):
        for h in range(H):
            n = int(pages[b, h])
            bt[b, h, :n] = perm[off:off + n]
            off += n
    return bt, total


def pool(total, P, D, fill=0xFF):
    """Pools whose unwritten bytes read as NaN (0xFFFF is a bf16 NaN)."""
    return [torch.full((total, P // 16, 10 * D), fill, dtype=torch.uint8) for _ in range(2)]


def check_append(k, v, lens, mask, P, D, seed, caps=None, table=None, **kw):
    """One append on the device and in the oracle: bytes, lengths, status."""
    import wgkv
    gen = torch.Generator().manual_seed(seed)
    B, T, H, _ = k.shape
    n_new = torch.full((B, H), T) if mask is None else mask.to(torch.bool).sum(2).cpu()
    bt, total = table_for(lens.clamp(min=0) + n_new, P, gen)
    if table is not None:
        bt = table(bt, total)
    if caps is not None:
        bt = bt[..., :caps].contiguous()
    kc, vc = pool(total, P, D)
    dk, dv = kc.to(DEV), vc.to(DEV)
    status = torch.zeros(1, dtype=I32, device=DEV)
    print(f"[kv4 append] k={tuple(k.shape)} {k.dtype} P={P} pages={total} table={tuple(bt.shape)}", flush=True)
    new = wgkv.kv4_append(k.to(DEV) if not k.is_cuda else k, v.to(DEV) if not v.is_cuda else v, dk, dv, bt.to(DEV),
                          lens.to(DEV, I32), g_mask=None if mask is None else mask.to(DEV), status=status, **kw)
    torch.cuda.synchronize()
    okc, ovc = kc.numpy(), vc.numpy()
    ref, lost = ok.append(k.double().cpu().numpy(), v.double().cpu().numpy(), okc, ovc, bt.numpy(), lens.numpy(),
                          None if mask is None else mask.bool().cpu().numpy())
    assert np.array_equal(new.cpu().numpy(), ref)
    assert int(status) == (3 if lost else 0)
    for got, want, what in ((dk, okc, "k"), (dv, ovc, "v")):
        diff = got.cpu().numpy() != want
        assert not diff.any(), f"{what}: {int(diff.sum())} bytes differ, first at {np.argwhere(diff)[0]}"
    return dk, dv, bt, new


def rows(gen, *shape, dtype=torch.bfloat16):
    x = torch.randn(*shape, generator=gen) * (1 + 3 * (torch.arange(shape[-1]) % 29 == 3)) + 0.5
    return x.to(dtype)


@pytest.mark.parametrize("D,P", [(64, 16), (64, 64), (128, 16), (128, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,kind", [(1, "all"), (3, "all"), (70, "all"), (64, "mask"), (131, "mask"), (40, "none")])
def test_append(D, P, dtype, T, kind):
    gen = torch.Generator().manual_seed(T * D + P)
    B, H = 2, 3
    k, v = rows(gen, B, T, H, D, dtype=dtype), rows(gen, B, T, H, D, dtype=dtype)
    lens = torch.tensor([[0, 1, 15], [16, 37, 130]], dtype=I32)
    mask = None
    if kind == "mask":
        mask = torch.rand(B, H, T, generator=gen) < torch.tensor([0.05, 0.4, 0.97])[None, :, None]
        mask[1, 0] = False
    elif kind == "none":
        mask = torch.zeros(B, H, T, dtype=torch.bool)
    check_append(k, v, lens, mask, P, D, seed=1)


@pytest.mark.parametrize("masked", [False, True])
def test_append_over_segments(masked):
    """Several counting segments, an odd row length (unaligned mask rows)."""
    gen = torch.Generator().manual_seed(9)
    B, T, H, D = 1, 8321, 2, 64
    k, v = rows(gen, B, T, H, D), rows(gen, B, T, H, D)
    mask = (torch.rand(B, H, T, generator=gen) < 0.08).to(torch.uint8) * 7 if masked else None
    if not masked:
        k, v = k[:, :4500], v[:, :4500]
    check_append(k, v, torch.tensor([[5, 0]], dtype=I32), mask, 16, D, seed=2)


@pytest.mark.parametrize("what", ["heads_first", "slice", "misaligned", "last_dim", "expanded", "mask_strided", "u8"])
def test_append_layouts(what):
    gen = torch.Generator().manual_seed(3)
    B, T, H, D = 2, 37, 2, 64
    k, v = rows(gen, B, T, H, D).to(DEV), rows(gen, B, T, H, D).to(DEV)
    mask = (torch.rand(B, H, T, generator=gen) < 0.5).to(DEV)
    if what == "heads_first":
        k = k.transpose(1, 2).contiguous().transpose(1, 2)
    elif what == "slice":
        big = torch.zeros(B, T + 2, 3 * H, D, dtype=torch.bfloat16, device=DEV)
        big[:, 1:-1, H:2 * H] = k
        k = big[:, 1:-1, H:2 * H]
    elif what == "misaligned":
        big = torch.zeros(B, T, H, D + 3, dtype=torch.bfloat16, device=DEV)
        big[..., 3:] = k
        k = big[..., 3:]
    elif what == "last_dim":
        v = v.transpose(2, 3).contiguous().transpose(2, 3)
    elif what == "expanded":
        k, v = k[:, :, :1].expand(B, T, H, D), v[:1].expand(B, T, H, D)
    elif what == "mask_strided":
        mask = mask.transpose(1, 2).contiguous().transpose(1, 2)
    else:
        mask = mask.to(torch.uint8) * 200
    check_append(k, v, torch.tensor([[0, 7], [18, 33]], dtype=I32), mask, 16, D, seed=4)


def test_append_borders_between_codes():
    """Values on and next to the borders between two codes fall on their
    side: exact multiples of the step (ties go to the even code), and fp32
    neighbours of them."""
    D = 64
    s, m = 0.25, 1.0
    ticks = m + s * np.arange(-7, 8)                     # the 15 borders, range 14 s of 15 s
    row = np.concatenate([[m - 7.5 * s, m + 7.5 * s], ticks, ticks])
    x32 = row.astype(np.float32)
    x32[2:17] = np.nextafter(x32[2:17], np.float32(np.inf))
    x32[17:] = np.nextafter(x32[17:], np.float32(-np.inf))
    for arr, dt in ((row, torch.bfloat16), (row, torch.float16), (x32, torch.float32)):
        x = torch.from_numpy(np.tile(arr, 2)).to(dt).view(1, 1, 1, D)
        assert np.array_equal(ok.quantise(x.double().numpy())[1].ravel(), [s, s])
        check_append(x, -x, torch.zeros(1, 1, dtype=I32), None, 16, D, seed=5)
    # a step whose fp32 rounding lies halfway between two bf16 values
    x = torch.linspace(-2.0 ** -26, 15 * (1 + 2.0 ** -8), 32)
    x[0], x[31] = -2.0 ** -26, 15 * (1 + 2.0 ** -8)
    assert ok.quantise(x.double().numpy())[1].item() == 1.0
    x = torch.cat([x, -x]).view(1, 1, 1, D)
    check_append(x, -x, torch.zeros(1, 1, dtype=I32), None, 16, D, seed=5)
    # tiny values beside large middles, and fp32 rows of wide dynamic range
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(1, 50, 2, D, generator=gen) * torch.exp(8 * torch.randn(1, 50, 2, D, generator=gen))
    check_append(x, x.flip(1), torch.zeros(1, 2, dtype=I32), None, 16, D, seed=5)


def test_append_special_values():
    D, T = 64, 12
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(1, T, 1, D, generator=gen)
    x[0, 0, 0, :32] = -2.5
    x[0, 1, 0, 3] = float("inf")
    x[0, 2, 0, 40] = float("nan")
    x[0, 3, 0, :32] = torch.linspace(-3e38, 3e38, 32)
    x[0, 4, 0, :32] = torch.linspace(0, 1e-40, 32)
    x[0, 5, 0] = 0.0
    x[0, 6, 0] = 3.4e38
    x[0, 7, 0, :32] = 100 + torch.linspace(-0.01, 0.01, 32)
    x[0, 8, 0, 5] = -float("inf")
    x[0, 9, 0] = 2.0 ** -120 * torch.randn(D, generator=gen)
    x[0, 10, 0, :32] = 3.38e38
    for dt in (torch.float32, torch.bfloat16):
        check_append(x.to(dt), -x.to(dt), torch.zeros(1, 1, dtype=I32), None, 16, D, seed=9)
    mask = torch.isfinite(x).all(-1).transpose(1, 2)  # what the mask leaves out may hold anything
    check_append(x, -x, torch.zeros(1, 1, dtype=I32), mask, 16, D, seed=9)


def test_append_without_room():
    """Tokens past the table and on pages outside the pool are dropped, the
    status is raised, lengths stop at the capacity; nothing else is touched."""
    gen = torch.Generator().manual_seed(10)
    k, v = rows(gen, 2, 70, 2, 64), rows(gen, 2, 70, 2, 64)
    lens = torch.tensor([[0, 30], [47, 500]], dtype=I32)
    _, _, _, new = check_append(k, v, lens, None, 16, 64, seed=11, caps=4)
    assert new.cpu().tolist() == [[64, 64], [64, 64]]

    def holes(bt, total):
        bt = bt.clone()
        bt[0, 0, 1] = -1
        bt[1, 0, 3] = total
        bt[1, 1, 0] = 2 ** 31 - 1
        return bt
    check_append(k, v, torch.tensor([[0, 30], [47, -3]], dtype=I32), None, 16, 64, seed=12, table=holes)


def test_append_nothing():
    k = torch.zeros(2, 0, 2, 64, dtype=torch.bfloat16)
    check_append(k, k.clone(), torch.tensor([[0, 5], [17, 2]], dtype=I32), None, 16, 64, seed=13)


@pytest.mark.parametrize("T", [1, 64, 200])
def test_append_writes_lengths_in_place(T):
    import wgkv
    gen = torch.Generator().manual_seed(T)
    k, v = rows(gen, 2, T, 3, 64).to(DEV), rows(gen, 2, T, 3, 64).to(DEV)
    lens = torch.tensor([[0, 3, 9], [33, 1, 16]], dtype=I32)
    bt, total = table_for(lens + T, 16, gen)
    a, b = [[t.to(DEV) for t in pool(total, 16, 64)] for _ in range(2)]
    sl = lens.to(DEV)
    new = wgkv.kv4_append(k, v, *a, bt.to(DEV), sl)
    assert torch.equal(sl.cpu(), lens)
    assert wgkv.kv4_append(k, v, *b, bt.to(DEV), sl, out=sl) is sl
    assert torch.equal(sl, new) and torch.equal(new.cpu(), lens + T)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def random_cache(gen, lens, P, D, spare=0):
    """A cache of random tokens written by the oracle's packer's rules (any
    codes, steps and middles), bytes past the lengths reading as NaN."""
    bt, total = table_for(lens, P, gen, spare)
    kc, vc = (x.numpy() for x in pool(total, P, D))
    rng = np.random.default_rng(int(torch.randint(1 << 30, (1,), generator=gen)))
    for b in range(lens.shape[0]):
        for h in range(lens.shape[1]):
            for p in range(int(lens[b, h])):
                pg = int(bt[b, h, p // P])
                for cache, keys in ((kc, True), (vc, False)):
                    ok.put(cache[pg, p % P // 16], p % 16, rng.integers(0, 16, D),
                           ok.bf16(rng.uniform(0.05, 0.4, D // 32)), ok.bf16(rng.normal(size=D // 32) * 0.3), keys)
    return kc, vc, bt


def oracle_read(kc, vc, bt, lens, n, starts):
    B, H = lens.shape
    D = kc.shape[2] // 10
    out = [np.zeros((B, n, H, D)), np.zeros((B, n, H, D))]
    for b in range(B):
        for h in range(H):
            ln, st = int(lens[b, h]), max(int(starts[b, h]), 0)
            for o, cache, keys in ((out[0], kc, True), (out[1], vc, False)):
                x = ok.values(*ok.rows(cache, bt[b, h].numpy(), ln, keys)) if ln else np.zeros((0, D))
                x = x[st:st + n]
                o[b, :x.shape[0], h] = x
    return [torch.from_numpy(o) for o in out]


@pytest.mark.parametrize("D,P", [(64, 16), (64, 32), (128, 16), (128, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_read(D, P, dtype):
    import wgkv
    gen = torch.Generator().manual_seed(D + P)
    lens = torch.tensor([[0, 1, 15], [64, 37, 130]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, P, D)
    dk, dv = torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV)
    for n, starts in [(130, None), (1, None), (200, None), (3, [[0, 0, 14], [61, 37, 127]]), (40, [[7, -3, 1], [2, 30, 99]])]:
        print(f"[kv4 read] D={D} P={P} {dtype} rows={n} starts={starts}", flush=True)
        st = None if starts is None else torch.tensor(starts, dtype=I32)
        got = wgkv.kv4_read(dk, dv, bt.to(DEV), lens.to(DEV), n, starts=None if st is None else st.to(DEV), dtype=dtype)
        want = oracle_read(kc, vc, bt, lens, n, torch.zeros_like(lens) if st is None else st)
        for g, w in zip(got, want):
            assert g.dtype == dtype and torch.equal(g.cpu(), w.float().to(dtype))


def test_read_out_tensors_and_bad_pages():
    import wgkv
    gen = torch.Generator().manual_seed(21)
    lens = torch.tensor([[40, 70]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 16, 64)
    dk, dv, dl = torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV), lens.to(DEV)
    ref = wgkv.kv4_read(dk, dv, bt.to(DEV), dl, 70)
    heads_first = [torch.zeros(1, 2, 70, 64, dtype=torch.bfloat16, device=DEV).transpose(1, 2) for _ in range(2)]
    odd = [torch.zeros(1, 70, 2, 67, dtype=torch.bfloat16, device=DEV)[..., 3:] for _ in range(2)]
    mixed = [heads_first[0].clone(), torch.zeros(1, 70, 2, 64, dtype=torch.bfloat16, device=DEV)]
    for out in (heads_first, odd, mixed):
        got = wgkv.kv4_read(dk, dv, bt.to(DEV), dl, 70, out=out)
        assert got[0] is out[0] and torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    bad = bt.clone()
    bad[0, 0, 1], bad[0, 1, 4] = kc.shape[0], -7
    got = wgkv.kv4_read(dk, dv, bad.to(DEV), dl, 70)
    for g, r in zip(got, ref):
        r = r.clone()
        r[0, 16:32, 0] = 0
        r[0, 64:, 1] = 0
        assert torch.equal(g, r)
    assert wgkv.kv4_read(dk, dv, bt.to(DEV), dl, 0)[0].shape == (1, 0, 2, 64)


def check_attend(q, kc, vc, bt, lens, scale, **kw):
    import wgkv
    print(f"[kv4 attend] q={tuple(q.shape)} pool={kc.shape} lens={lens.flatten().tolist()[:8]}", flush=True)
    got = wgkv.paged_decode_attn_kv4(q.to(DEV), torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV),
                                     lens.to(DEV), bt.to(DEV), scale, **kw)
    torch.cuda.synchronize()
    want, bound = ok.attend(q[:, 0].double().numpy(), kc, vc, bt.numpy(), lens.numpy(), scale)
    err = np.abs(got[:, 0].double().cpu().numpy() - want)
    assert (err <= bound).all(), f"worst error / bound {np.nanmax(err / bound)}, nan {int(np.isnan(err).sum())}"
    return got


@pytest.mark.parametrize("D,P", [(64, 16), (64, 64), (128, 16), (128, 32)])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 7, 8])
def test_attend_head_groups(D, P, G):
    gen = torch.Generator().manual_seed(G * D + P)
    lens = torch.tensor([[0, 1, 33], [16, 95, 128]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, P, D)
    q = torch.randn(2, 1, 3 * G, D, generator=gen).to(torch.bfloat16)
    check_attend(q, kc, vc, bt, lens, D ** -0.5)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 511, 513])
def test_attend_lengths(n):
    gen = torch.Generator().manual_seed(n)
    lens = torch.tensor([[n, max(0, n - 1)]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 16, 64, spare=2)
    q = torch.randn(1, 1, 8, 64, generator=gen).to(torch.bfloat16)
    check_attend(q, kc, vc, bt, lens, 64 ** -0.5)


def device_cache(lens, P, D, seed, total=None):
    """A cache filled on the device by kv4_append; (kc, vc, table)."""
    import wgkv
    gen = torch.Generator().manual_seed(seed)
    bt, n = table_for(lens, P, gen)
    kc, vc = (t.to(DEV) for t in pool(n, P, D))
    T = int(lens.max())
    B, H = lens.shape
    g = torch.Generator(device=DEV).manual_seed(seed)
    k, v = (torch.randn(B, T, H, D, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    mask = torch.arange(T)[None, None] < lens[..., None]
    new = wgkv.kv4_append(k, v, kc, vc, bt.to(DEV), torch.zeros_like(lens).to(DEV), g_mask=mask.to(DEV))
    assert torch.equal(new.cpu(), lens)
    return kc, vc, bt


@pytest.mark.parametrize("B,H,G,D,lens", [
    (1, 1, 4, 128, [4097]),
    (1, 2, 8, 128, [3000, 17]),
    (1, 1, 8, 64, [5003]),
    (2, 20, 2, 64, "ragged"),       # 40 heads
    (3, 30, 4, 128, "short"),       # 90 heads
])
def test_attend_split_over_workgroups(B, H, G, D, lens):
    """Heads cut over many workgroups, among others of every length."""
    gen = torch.Generator().manual_seed(B * H + D)
    if lens == "ragged":
        ln = torch.randint(0, 900, (B, H), generator=gen, dtype=I32)
        ln[0, 3], ln[1, 7] = 0, 2600
    elif lens == "short":
        ln = torch.randint(0, 70, (B, H), generator=gen, dtype=I32)
        ln[2, 29] = 1500
    else:
        ln = torch.tensor(lens, dtype=I32).view(B, H)
    kc, vc, bt = device_cache(ln, 16, D, seed=B + H)
    q = torch.randn(B, 1, H * G, D, generator=gen).to(torch.bfloat16)
    check_attend(q, kc.cpu().numpy(), vc.cpu().numpy(), bt, ln, D ** -0.5)


def test_attend_many_heads():
    """2048 heads: the most the call takes; lengths 0 to 40."""
    gen = torch.Generator().manual_seed(31)
    ln = torch.randint(0, 41, (64, 32), generator=gen, dtype=I32)
    kc, vc, bt = device_cache(ln, 16, 64, seed=32)
    q = torch.randn(64, 1, 32, 64, generator=gen).to(torch.bfloat16)
    check_attend(q, kc.cpu().numpy(), vc.cpu().numpy(), bt, ln, 0.125)


@pytest.mark.parametrize("what", ["large_scores", "one_dominant", "zero_scale", "negative_scale", "equal"])
def test_attend_scores(what):
    gen = torch.Generator().manual_seed(41)
    lens = torch.tensor([[200, 77]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 16, 64)
    q = torch.randn(1, 1, 4, 64, generator=gen)
    scale = 0.125
    if what == "large_scores":
        q = q * 40
    elif what == "one_dominant":
        q = q * 0.01
        c, s, m = ok.get(kc[int(bt[0, 0, 11]), 0], 5, 64, True)
        q[0, 0, :2] = torch.from_numpy(ok.values(c, s, m)).float() * 30
    elif what == "zero_scale":
        scale = 0.0
    elif what == "negative_scale":
        scale = -0.7
    else:
        q = torch.zeros_like(q)
    check_attend(q.to(torch.bfloat16), kc, vc, bt, lens, scale)


def test_attend_nan_in_a_head_stays_there():
    """A stored NaN makes its own head's output NaN and no other's."""
    import wgkv
    gen = torch.Generator().manual_seed(43)
    lens = torch.tensor([[50, 50]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 16, 64)
    q = torch.randn(1, 1, 4, 64, generator=gen).to(torch.bfloat16)
    ok.put(kc[int(bt[0, 1, 2]), 0], 3, np.zeros(64, np.int64), np.array([np.nan, 0.1]), np.array([np.nan, 0.0]), True)
    got = wgkv.paged_decode_attn_kv4(q.to(DEV), torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV),
                                     lens.to(DEV), bt.to(DEV), 0.125).cpu()
    want, bound = ok.attend(q[:, 0].double().numpy(), kc, vc, bt.numpy(), torch.tensor([[50, 0]]).numpy(), 0.125)
    assert (np.abs(got[0, 0, :2].double().numpy() - want[0, :2]) <= bound[0, :2]).all()
    assert torch.isnan(got[0, 0, 2:]).all()


def test_attend_clamps_lengths_and_pages():
    gen = torch.Generator().manual_seed(44)
    lens = torch.tensor([[64, 30, 16]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 16, 64)
    q = torch.randn(1, 1, 6, 64, generator=gen).to(torch.bfloat16)
    for x in (kc, vc):  # the pages that clamped ids reach hold numbers
        x[0] = x[int(bt[0, 0, 1])]
        x[-1] = x[int(bt[0, 1, 0])]
    bt = bt.clone()
    bt[0, 0, 2], bt[0, 1, 0] = -5, 2 ** 31 - 1
    check_attend(q, kc, vc, bt[..., :4], torch.tensor([[2 ** 31 - 1, 30, -9]], dtype=I32), 0.125)


@pytest.mark.parametrize("what", ["q_slice", "q_misaligned", "out", "out_misaligned", "tables"])
def test_attend_layouts(what):
    import wgkv
    gen = torch.Generator().manual_seed(45)
    lens = torch.tensor([[64, 30], [7, 16]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 16, 64)
    dk, dv = torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV)
    q = torch.randn(2, 1, 4, 64, generator=gen).to(torch.bfloat16).to(DEV)
    sl, tb, out = lens.to(DEV), bt.to(DEV), None
    ref = wgkv.paged_decode_attn_kv4(q, dk, dv, sl, tb, 0.125)
    if what == "q_slice":
        q = torch.cat([q, q, q], 2)[:, :, 4:8]
    elif what == "q_misaligned":
        q = torch.nn.functional.pad(q, (1, 2))[..., 1:-2]
    elif what == "out":
        out = torch.zeros(2, 1, 12, 64, dtype=torch.bfloat16, device=DEV)[:, :, 4:8]
    elif what == "out_misaligned":
        out = torch.zeros(2, 1, 4, 65, dtype=torch.bfloat16, device=DEV)[..., 1:]
    else:
        sl = sl.t().contiguous().t()
        tb = torch.stack([tb, tb], -1)[..., 0]
    got = wgkv.paged_decode_attn_kv4(q, dk, dv, sl, tb, 0.125, out=out)
    assert torch.equal(got, ref) and (out is None or got is out)


def test_pool_beyond_32_bits():
    """Pages past 4 GiB of a pool, and single rows there."""
    import wgkv
    D, P, n = 128, 64, 900_000  # 4.6 GB each
    kc, vc = (torch.empty(n, P // 16, 10 * D, dtype=torch.uint8, device=DEV) for _ in range(2))
    gen = torch.Generator().manual_seed(51)
    T = 100
    k, v = rows(gen, 1, T, 1, D), rows(gen, 1, T, 1, D)
    q = torch.randn(1, 1, 4, D, generator=gen).to(torch.bfloat16)
    small = [x.numpy() for x in pool(2, P, D)]
    ok.append(k.double().numpy(), v.double().numpy(), *small, np.array([[[0, 1]]]), np.zeros((1, 1), np.int64))
    bt = torch.tensor([[[n - 1, n - 7]]], dtype=I32, device=DEV)
    sl = wgkv.kv4_append(k.to(DEV), v.to(DEV), kc, vc, bt, torch.zeros(1, 1, dtype=I32, device=DEV))
    assert torch.equal(kc[n - 1].cpu(), torch.from_numpy(small[0][0]))
    want = oracle_read(*small, torch.tensor([[[0, 1]]]), torch.tensor([[T]]), T, torch.zeros(1, 1))
    for g, w in zip(wgkv.kv4_read(kc, vc, bt, sl, T), want):
        assert torch.equal(g.cpu(), w.to(torch.bfloat16))
    got = wgkv.paged_decode_attn_kv4(q.to(DEV), kc, vc, sl, bt, D ** -0.5)
    ref, bound = ok.attend(q[:, 0].double().numpy(), *small, np.array([[[0, 1]]]), np.array([[T]]), D ** -0.5)
    assert (np.abs(got[:, 0].double().cpu().numpy() - ref) <= bound).all()


def test_prompt_then_decode_steps():
    """The operators as a decoder uses them: a gated prompt is appended, then
    each step appends its token and attends; the cache read back at the end
    is the oracle's."""
    import wgkv
    gen = torch.Generator().manual_seed(61)
    B, H, G, D, P, S, steps = 2, 2, 4, 128, 16, 150, 5
    k, v = rows(gen, B, S, H, D), rows(gen, B, S, H, D)
    mask = torch.rand(B, H, S, generator=gen) < 0.4
    mask[0, 1] = False
    n = mask.sum(2) + steps
    bt, total = table_for(n, P, gen)
    kc, vc = (x.numpy() for x in pool(total, P, D))
    dk, dv = torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV)
    sl = torch.zeros(B, H, dtype=I32, device=DEV)
    ref, _ = ok.append(k.double().numpy(), v.double().numpy(), kc, vc, bt.numpy(), np.zeros((B, H), np.int64), mask.numpy())
    wgkv.kv4_append(k.to(DEV), v.to(DEV), dk, dv, bt.to(DEV), sl, g_mask=mask.to(DEV), out=sl)
    for i in range(steps):
        k1, v1 = rows(gen, B, 1, H, D), rows(gen, B, 1, H, D)
        q = torch.randn(B, 1, H * G, D, generator=gen).to(torch.bfloat16)
        ref, _ = ok.append(k1.double().numpy(), v1.double().numpy(), kc, vc, bt.numpy(), ref)
        wgkv.kv4_append(k1.to(DEV), v1.to(DEV), dk, dv, bt.to(DEV), sl, out=sl)
        got = wgkv.paged_decode_attn_kv4(q.to(DEV), dk, dv, sl, bt.to(DEV), D ** -0.5)
        want, bound = ok.attend(q[:, 0].double().numpy(), kc, vc, bt.numpy(), ref, D ** -0.5)
        assert (np.abs(got[:, 0].double().cpu().numpy() - want) <= bound).all(), i
    assert np.array_equal(sl.cpu().numpy(), ref)
    for g, w in zip(wgkv.kv4_read(dk, dv, bt.to(DEV), sl, int(n.max()), dtype=torch.float32),
                    oracle_read(kc, vc, bt, torch.from_numpy(ref), int(n.max()), torch.zeros(B, H))):
        assert torch.equal(g.cpu(), w.float())


def test_captured_decode_step():
    """Two captured steps (append, attend) replayed in turn with eager calls
    between them: each replay continues the same caches."""
    import wgkv
    gen = torch.Generator().manual_seed(71)
    B, H, G, D, P, S, steps = 1, 4, 4, 128, 16, 600, 6
    lens = torch.tensor([[S, 30, 1, 257]], dtype=I32)
    kc, vc, bt = device_cache(lens, P, D, seed=72)
    width = int((lens.max() + 2 * steps + P - 1) // P)
    total = kc.shape[0]
    full = torch.full((B, H, width), -1, dtype=I32)
    full[..., :bt.shape[2]] = bt
    for h in range(H):  # pages for the steps to come
        for j in range(width):
            if full[0, h, j] < 0:
                full[0, h, j] = total
                total += 1
    kc, vc = (torch.cat([x, torch.zeros(total - x.shape[0], *x.shape[1:], dtype=torch.uint8, device=DEV)]) for x in (kc, vc))
    full = full.to(DEV)

    def state():
        return kc.clone(), vc.clone(), lens.to(DEV)
    ins = [tuple(torch.randn(B, 1, n, D, generator=gen).to(torch.bfloat16).to(DEV) for n in (H, H, H * G))
           for _ in range(2 * steps)]
    ea, ga, gb = state(), state(), state()

    def step(st, k1, v1, q):
        wgkv.kv4_append(k1, v1, st[0], st[1], full, st[2], out=st[2])
        return wgkv.paged_decode_attn_kv4(q, st[0], st[1], st[2], full, D ** -0.5)
    stat = [[torch.zeros_like(t) for t in ins[0]] for _ in range(2)]
    warm = state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, *ins[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for st, x in ((ga, stat[0]), (gb, stat[1])):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(st, *x))
        graphs.append(g)
    for i in range(steps):
        want = step(ea, *ins[i])
        for g, x, o in zip(graphs, stat, outs):
            for d, s in zip(x, ins[i]):
                d.copy_(s)
            g.replay()
            assert torch.equal(o, want), i
        torch.cuda.synchronize()
    for st in (ga, gb):
        assert all(torch.equal(x, y) for x, y in zip(st, ea))
    # both graphs at once, on streams of their own
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for i in range(steps, 2 * steps):
        want = step(ea, *ins[i])
        for x in stat:
            for d, s in zip(x, ins[i]):
                d.copy_(s)
        torch.cuda.synchronize()
        for g, s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), i


def test_calls_on_two_streams_at_once():
    import wgkv
    gen = torch.Generator().manual_seed(81)
    ln = torch.randint(500, 3000, (2, 8), generator=gen, dtype=I32)
    kc, vc, bt = device_cache(ln, 16, 128, seed=82)
    sl, tb = ln.to(DEV), bt.to(DEV)
    qs = [torch.randn(2, 1, 32, 128, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2)]
    refs = [wgkv.paged_decode_attn_kv4(q, kc, vc, sl, tb, 0.09) for q in qs]
    rk = wgkv.kv4_read(kc, vc, tb, sl, 600)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [[], []]
    for i in range(20):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[j].append(wgkv.paged_decode_attn_kv4(qs[j], kc, vc, sl, tb, 0.09))
                if i % 7 == 0:
                    got = wgkv.kv4_read(kc, vc, tb, sl, 600)
                    outs[j].append(got)
    torch.cuda.synchronize()
    for j in range(2):
        for o in outs[j]:
            if isinstance(o, tuple):
                assert torch.equal(o[0], rk[0]) and torch.equal(o[1], rk[1])
            else:
                assert torch.equal(o, refs[j])


def test_dispatcher_operators_run_the_kernels():
    import wgkv
    gen = torch.Generator().manual_seed(91)
    lens = torch.tensor([[70, 33]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 32, 128)
    dk, dv, sl, tb = torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV), lens.to(DEV), bt.to(DEV)
    q = torch.randn(1, 1, 8, 128, generator=gen).to(torch.bfloat16).to(DEV)
    assert torch.equal(torch.ops.wgkv.paged_decode_attn_kv4(q, dk, dv, sl, tb, 0.1),
                       wgkv.paged_decode_attn_kv4(q, dk, dv, sl, tb, 0.1))
    for a, b in zip(torch.ops.wgkv.kv4_read(dk, dv, tb, sl, 40, dtype=torch.float32),
                    wgkv.kv4_read(dk, dv, tb, sl, 40, dtype=torch.float32)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("units", [16, 17, 32, 33])
def test_attend_page_windows(units):
    """Ranges that end with or just behind a window of page ids (16 units of
    64 tokens): one head on one workgroup's waves, many units each."""
    import wgkv
    ln = torch.full((64, 32), 1, dtype=I32)  # 2048 heads fill the line's other ranges
    ln[5, 7] = units * 64
    ln[63, 31] = units * 64 - 40
    kc, vc, bt = device_cache(ln, 64, 64, seed=units)
    gen = torch.Generator().manual_seed(units)
    q = torch.randn(64, 1, 32, 64, generator=gen).to(torch.bfloat16)
    check_attend(q, kc.cpu().numpy(), vc.cpu().numpy(), bt, ln, 0.125)
    # the same heads alone, whole ranges of many units per wave
    long = torch.full((8, 8), units * 64 * 4, dtype=I32)
    kc, vc, bt = device_cache(long, 64, 64, seed=units + 1)
    q = torch.randn(8, 1, 32, 64, generator=gen).to(torch.bfloat16).to(DEV)
    sl, tb = long.to(DEV), bt.to(DEV)
    got = wgkv.paged_decode_attn_kv4(q, kc, vc, sl, tb, 0.125)
    k, v = wgkv.kv4_read(kc, vc, tb, sl, units * 256, dtype=torch.float32)
    k, v = (x.cpu().double().transpose(1, 2).repeat_interleave(4, 1) for x in (k, v))
    p = torch.softmax((q.cpu().double().transpose(1, 2) @ k.transpose(2, 3)) * 0.125, -1)
    want = (p @ v).transpose(1, 2)
    # half a bf16 step, 2^-8, of what the codes add (a group's middle is that
    # of its read values, whose ends are codes 0 and 15) and of the output;
    # fp32 sums: 32 accumulations of codes offset by 143 steps of at most 0.5
    # between two corrections, and as much for their offset: 2 * 32 * 2^-24 *
    # 143 * 0.5 = 2.8e-4
    g = v.view(*v.shape[:-1], 2, 32)
    spread = (g - (g.amax(-1, keepdim=True) + g.amin(-1, keepdim=True)) / 2).abs().view_as(v)
    bound = 2.0 ** -8 * ((p @ spread).transpose(1, 2) + want.abs()) + 2.8e-4
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("T,masked", [(17161, True), (16384, True), (5000, False)])
def test_append_long_prompts_in_place(T, masked):
    """Prompts of several counting segments, their lengths written apart and
    in place; the mask's rows start at any byte."""
    import wgkv
    gen = torch.Generator().manual_seed(T)
    B, H, D, P = 1, 3, 64, 32
    k, v = rows(gen, B, T, H, D), rows(gen, B, T, H, D)
    lens = torch.tensor([[5, 0, 77]], dtype=I32)
    mask = torch.rand(B, H, T, generator=gen) < 0.05 if masked else None
    if masked:
        mask[0, 1, 4090:12300] = False
        mask[0, 2, T - 300:] = True
    dk, dv, bt, new = check_append(k, v, lens, mask, P, D, seed=3)
    b = [t.to(DEV) for t in pool(dk.shape[0], P, D)]
    sl = lens.to(DEV)
    wgkv.kv4_append(k.to(DEV), v.to(DEV), *b, bt.to(DEV), sl, g_mask=None if mask is None else mask.to(DEV), out=sl)
    assert torch.equal(sl, new) and torch.equal(b[0], dk) and torch.equal(b[1], dv)


def test_append_lengths_beside_each_other():
    """Lengths read from one half of an array and written to the other, and
    lengths of one row for every sequence."""
    import wgkv
    gen = torch.Generator().manual_seed(103)
    k, v = rows(gen, 2, 300, 3, 64).to(DEV), rows(gen, 2, 300, 3, 64).to(DEV)
    lens = torch.tensor([[4, 0, 19]], dtype=I32).expand(2, 3)
    bt, total = table_for(lens + 300, 16, gen)
    both = torch.cat([lens, torch.full_like(lens, -7)], 1).to(DEV)
    a, b = [[t.to(DEV) for t in pool(total, 16, 64)] for _ in range(2)]
    wgkv.kv4_append(k, v, *a, bt.to(DEV), both[:, :3], out=both[:, 3:])
    new = wgkv.kv4_append(k, v, *b, bt.to(DEV), lens[:1].to(DEV).expand(2, 3))
    assert torch.equal(both[:, :3].cpu(), lens) and torch.equal(both[:, 3:], new) and torch.equal(new.cpu(), lens + 300)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_overlapping_outputs_are_refused():
    import wgkv
    from wgkv import _lib
    gen = torch.Generator().manual_seed(105)
    lens = torch.tensor([[20, 3], [0, 9]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 16, 64)
    dk, dv, tb = torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV), bt.to(DEV)
    k = rows(gen, 2, 4, 2, 64).to(DEV)
    buf = torch.zeros(3, 2, dtype=I32, device=DEV)
    for sl, out in [(buf[:2], buf[1:]), (buf[1:], buf[:2]), (buf[:2], torch.zeros(1, 2, dtype=I32, device=DEV).expand(2, 2))]:
        with pytest.raises(_lib.WGKVError):
            wgkv.kv4_append(k, k.clone(), dk, dv, tb, sl, out=out)
    sl = lens.to(DEV)
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(_lib.WGKVError):
        wgkv.paged_decode_attn_kv4(q, dk, dv, sl, tb, 0.1, out=q[:1].expand(2, 1, 4, 64))
    one = torch.zeros(2, 2, 1, 8, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(_lib.WGKVError):
        wgkv.kv4_read(dk, dv, tb, sl, 8, out=tuple(one.transpose(2, 3).expand(2, 2, 8, 2, 64)))
    assert torch.equal(dk.cpu(), torch.from_numpy(kc)) and not buf.any()


def test_captured_prompt_append():
    """A gated prompt's append of two launches, its scratch the graph's."""
    import wgkv
    gen = torch.Generator().manual_seed(107)
    B, T, H, D, P = 1, 16500, 2, 64, 32
    k, v = rows(gen, B, T, H, D).to(DEV), rows(gen, B, T, H, D).to(DEV)
    masks = [(torch.rand(B, H, T, generator=gen) < p).to(torch.uint8).to(DEV) for p in (0.02, 0.3, 0.1)]
    lens = torch.tensor([[9, 100]], dtype=I32, device=DEV)
    bt, total = table_for(torch.full((B, H), 3 * T), P, gen)
    tb = bt.to(DEV)
    ea, ga = ([t.to(DEV) for t in pool(total, P, D)] + [lens.clone()] for _ in range(2))
    m = masks[0].clone()

    def step(st, mask):
        wgkv.kv4_append(k, v, st[0], st[1], tb, st[2], g_mask=mask, out=st[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in ga], m)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(ga, m)
    for mask in masks:
        step(ea, mask)
        m.copy_(mask)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(ea, ga))


@pytest.mark.parametrize("B,H,G,D", [(3, 30, 8, 128), (7, 11, 5, 128), (9, 13, 3, 64)])
def test_attend_many_heads_of_wide_groups(B, H, G, D):
    gen = torch.Generator().manual_seed(B * G)
    ln = torch.randint(0, 90, (B, H), generator=gen, dtype=I32)
    ln[0, 0], ln[B - 1, H - 1], ln[1, 2] = 0, 2100, 900
    kc, vc, bt = device_cache(ln, 32, D, seed=B + H)
    q = torch.randn(B, 1, H * G, D, generator=gen).to(torch.bfloat16)
    check_attend(q, kc.cpu().numpy(), vc.cpu().numpy(), bt, ln, D ** -0.5)


def test_attend_nothing_anywhere():
    """No head has a token: zeros, whatever the pages and the table hold."""
    import wgkv
    for B, H, G, D in [(1, 1, 1, 64), (2, 3, 8, 128), (40, 5, 2, 64)]:
        kc, vc = (t.to(DEV) for t in pool(2, 16, D))
        bt = torch.full((B, H, 1), -1, dtype=I32, device=DEV)
        q = torch.full((B, 1, H * G, D), float("nan"), dtype=torch.bfloat16, device=DEV)
        out = torch.full_like(q, 3.0)
        for n in (0, -5):
            sl = torch.full((B, H), n, dtype=I32, device=DEV)
            assert not wgkv.paged_decode_attn_kv4(q, kc, vc, sl, bt, 0.1, out=out).any()


def test_attend_nan_in_a_query_stays_there():
    import wgkv
    gen = torch.Generator().manual_seed(109)
    lens = torch.tensor([[700, 33]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 16, 128)
    args = (torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV), lens.to(DEV), bt.to(DEV), 0.09)
    for G in (4, 7):
        q = torch.randn(1, 1, 2 * G, 128, generator=gen).to(torch.bfloat16).to(DEV)
        want, bound = ok.attend(q[:, 0].double().cpu().numpy(), kc, vc, bt.numpy(), lens.numpy(), 0.09)
        for bad in (0, G + 2):
            x = q.clone()
            x[0, 0, bad, 77] = float("nan")
            got = wgkv.paged_decode_attn_kv4(x, *args)[:, 0].double().cpu().numpy()
            keep = [i for i in range(2 * G) if i != bad]
            assert (np.abs(got - want) <= bound)[:, keep].all() and np.isnan(got[:, bad]).all()


def test_attend_scales_with_its_values():
    """Steps and middles of the values times a power of two: the output times
    the same, to the last bit (nothing under- or overflows on the way)."""
    import wgkv
    gen = torch.Generator().manual_seed(111)
    lens = torch.tensor([[1500, 70]], dtype=I32)
    P, D = 16, 64
    kc, vc, bt = random_cache(gen, lens, P, D)
    q = (torch.randn(1, 1, 8, D, generator=gen) * 0.5).to(torch.bfloat16).to(DEV)
    sl, tb, dk = lens.to(DEV), bt.to(DEV), torch.from_numpy(kc).to(DEV)
    ref = wgkv.paged_decode_attn_kv4(q, dk, torch.from_numpy(vc).to(DEV), sl, tb, 0.125)
    for e in (96, -60):
        x = torch.from_numpy(vc.copy())
        pairs = x[..., 8 * D:].contiguous().view(torch.bfloat16)
        x[..., 8 * D:] = (pairs.float() * 2.0 ** e).to(torch.bfloat16).view(torch.uint8)
        got = wgkv.paged_decode_attn_kv4(q, dk, x.to(DEV), sl, tb, 0.125)
        assert torch.equal(got.float(), ref.float() * 2.0 ** e)


def test_append_borders_of_the_smallest_steps():
    """The same at the least step, 2^-126, where neighbours of a border lie
    2^-149 (fp32) and 2^-133 (bf16) from it."""
    D = 64
    for s in (2.0 ** -126, 1.5 * 2.0 ** -126):
        for m in (0.0, 2.0 ** -122):
            ticks = m + s * np.arange(-7, 8)
            for dt, least in ((torch.float32, 2.0 ** -149), (torch.bfloat16, 2.0 ** -133)):
                rows_ = [np.concatenate([[m - 7.5 * s, m + 7.5 * s], ticks + e * least, ticks]) for e in (-1, 0, 1)]
                x = torch.from_numpy(np.concatenate([*rows_, rows_[0]]).reshape(2, D)).to(dt).view(1, 2, 1, D)
                want = ok.quantise(x.double().numpy())[1]
                assert np.isfinite(want).all() and (want > 0).all()
                check_append(x, -x, torch.zeros(1, 1, dtype=I32), None, 16, D, seed=7)


@pytest.mark.parametrize("B,H,G,D", [(64, 1, 2, 64), (5, 13, 1, 128), (4, 64, 4, 128), (257, 1, 3, 64), (5, 60, 8, 128)])
def test_attend_heads_per_lane(B, H, G, D):
    """64, 65, 256, 257 and 300 heads: 1 to 5 of them per lane of the line,
    empty ones in all places, a long one among the last."""
    gen = torch.Generator().manual_seed(B + H)
    ln = torch.randint(0, 70, (B, H), generator=gen, dtype=I32)
    ln[torch.rand(B, H, generator=gen) < 0.4] = 0
    ln.view(-1)[-2] = 1700
    kc, vc, bt = device_cache(ln, 16, D, seed=B * H)
    q = torch.randn(B, 1, H * G, D, generator=gen).to(torch.bfloat16)
    got = check_attend(q, kc.cpu().numpy(), vc.cpu().numpy(), bt, ln, D ** -0.5)
    assert not got.view(B, H, G * D)[(ln == 0).to(DEV)].any()


@pytest.mark.parametrize("extra", [0, 1, 63, 65, 129, 500])
def test_attend_uneven_ranges(extra):
    """Lines of a few units more than the workgroups and waves have ranges
    for: the first ranges are a unit longer than the others."""
    gen = torch.Generator().manual_seed(extra)
    units = 1024 + 3 * extra  # 256 workgroups of 4 units, and some
    ln = torch.tensor([[units * 64 // 4 - 640, units * 64 // 4 + 640 - 63, 70, units * 64 // 2 - 100]], dtype=I32)
    kc, vc, bt = device_cache(ln, 64, 64, seed=extra)
    q = torch.randn(1, 1, 8, 64, generator=gen).to(torch.bfloat16)
    check_attend(q, kc.cpu().numpy(), vc.cpu().numpy(), bt, ln, 0.125)


def test_captured_calls_share_one_scratch():
    """Graphs of several attention calls, on one stream and forked: a capture
    clears its scratch once per stream, whatever the calls' sizes, and no two
    captures share it."""
    import wgkv
    from wgkv import kv4
    gen = torch.Generator().manual_seed(121)
    ln = torch.tensor([[900, 3000, 0, 77]], dtype=I32)
    kc, vc, bt = device_cache(ln, 16, 128, seed=122)
    sl, tb = ln.to(DEV), bt.to(DEV)
    qs = [torch.randn(1, 1, 4 * g, 128, generator=gen).to(torch.bfloat16).to(DEV) for g in (1, 4, 2, 8, 8, 3)]
    want = [wgkv.paged_decode_attn_kv4(q, kc, vc, sl, tb, 0.09) for q in qs]
    torch.cuda.synchronize()
    graphs, seen = [], []
    fork = torch.cuda.Stream()
    for forked in (False, True, False):
        g, outs = torch.cuda.CUDAGraph(), []
        with torch.cuda.graph(g):
            main = torch.cuda.current_stream()
            for i, q in enumerate(qs):
                if forked and i == 1:
                    fork.wait_stream(main)
                    with torch.cuda.stream(fork):
                        outs.append(wgkv.paged_decode_attn_kv4(q, kc, vc, sl, tb, 0.09))
                        seen.append(kv4._captured[(0, fork.cuda_stream)])
                    main.wait_stream(fork)
                else:
                    outs.append(wgkv.paged_decode_attn_kv4(q, kc, vc, sl, tb, 0.09))
                seen.append(kv4._captured[(0, main.cuda_stream)])
        graphs.append((g, outs))
    ids = [i for i, _ in seen]
    assert len(set(ids)) == 3 and 0 not in ids
    # of the sizes G = 1, 4, 2, 8, 8, 3 only 1, 4 and 8 asked for more
    assert len({ws.data_ptr() for i, ws in seen if i == ids[0]}) == 3
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for (g, outs), s in zip(graphs, streams):
            for o in outs:
                o.fill_(9.0)
        torch.cuda.synchronize()
        for (g, outs), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = wgkv.paged_decode_attn_kv4(qs[1], kc, vc, sl, tb, 0.09)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[1])
        for _, outs in graphs:
            assert all(torch.equal(o, w) for o, w in zip(outs, want))


def minus_infinity_case(D, G, dead, n, seed):
    """One sequence of two heads whose first ``dead`` tokens (whole pages) have
    keys that every query of ones scores below the least fp32 number, before
    ``n`` ordinary ones: (q, kc, vc, table, lens, pages to skip)."""
    P = 16
    gen = torch.Generator().manual_seed(seed)
    lens = torch.tensor([[dead + n, dead + max(n - 30, 0)]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, P, D)
    for h in range(2):
        for p in range(dead):  # constant rows: step 0, -1e37 in every place
            ok.put(kc[int(bt[0, h, p // P]), 0], p % P, np.zeros(D, np.int64), np.zeros(D // 32), ok.bf16(np.full(D // 32, -1e37)), True)
    q = torch.randn(1, 1, 2 * G, D, generator=gen) * 0.1 + 1
    return q.to(torch.bfloat16), kc, vc, bt, lens, dead // P


@pytest.mark.parametrize("D,G", [(64, 8), (128, 4), (128, 7)])
@pytest.mark.parametrize("dead,n", [(16, 40), (64, 300), (320, 70), (1600, 33)])
def test_attend_scores_of_minus_infinity(D, G, dead, n):
    """Tokens whose score falls below fp32's range weigh nothing, wherever
    they stand: among a half's others, alone in a wave's range, in a piece."""
    import wgkv
    q, kc, vc, bt, lens, skip = minus_infinity_case(D, G, dead, n, seed=D + G + dead)
    want, bound = ok.attend(q[:, 0].double().numpy(), kc, vc, bt[..., skip:].numpy(), (lens - dead).numpy(), 0.125)
    dk, dv = torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV)
    print(f"[kv4 attend -inf] D={D} G={G} dead={dead} n={n}", flush=True)
    got = wgkv.paged_decode_attn_kv4(q.to(DEV), dk, dv, lens.to(DEV), bt.to(DEV), 0.125)
    assert (np.abs(got[:, 0].double().cpu().numpy() - want) <= bound).all()
    # scores that only the scale takes there: -1e37 * sum q is 1000 times too small
    x = (q.float() / 1000).to(torch.bfloat16)
    want, bound = ok.attend(x[:, 0].double().numpy(), kc, vc, bt[..., skip:].numpy(), (lens - dead).numpy(), 900.0)
    got = wgkv.paged_decode_attn_kv4(x.to(DEV), dk, dv, lens.to(DEV), bt.to(DEV), 900.0)
    assert (np.abs(got[:, 0].double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("dead", [16, 400])
def test_attend_only_scores_of_minus_infinity(dead):
    """No token left with any weight: zeros, as of a head without tokens."""
    import wgkv
    q, kc, vc, bt, lens, _ = minus_infinity_case(128, 4, dead, 0, seed=dead)
    got = wgkv.paged_decode_attn_kv4(q.to(DEV), torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV),
                                     lens.to(DEV), bt.to(DEV), 0.125)
    assert not got.any()


def test_append_middles_of_subnormal_groups():
    """fp32 groups below 2^-126, whose halves fp32 does not hold: middles next
    to a border between two bf16 values, and any others."""
    D, T = 64, 512
    unit = 2.0 ** -149  # of fp32; a bf16 unit there is 2^16 of them
    rng = np.random.default_rng(131)
    mid = rng.integers(1, 120, (1, T, 2, D // 32, 1)) * 2 ** 16 + 2 ** 15
    odd = np.stack([mid + rng.integers(-2, 3, mid.shape) for _ in range(2)])  # the ends: hi + lo odd in half of them
    pick = rng.integers(0, 2, (2, 1, T, 2, D // 32, 32))
    near = np.where(pick == 1, odd[0], odd[1])
    near[..., :1], near[..., 1:2] = odd[0], odd[1]
    wide = rng.integers(-2 ** 23 + 1, 2 ** 23, near.shape)
    for x in (near, wide):
        k, v = (torch.from_numpy((y * unit).reshape(1, T, 2, D)).float() for y in x)
        assert np.array_equal(k.double().numpy(), (x[0] * unit).reshape(1, T, 2, D))
        check_append(k, -v, torch.zeros(1, 2, dtype=I32), None, 16, D, seed=133)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_read_of_subnormal_values(dtype):
    """Middles below 2^-126 and, for fp16, values below 2^-14."""
    import wgkv
    gen = torch.Generator().manual_seed(137)
    x = torch.randn(1, 60, 1, 64, generator=gen)
    x = x * torch.tensor([2.0 ** -6, 2.0 ** -14, 2.0 ** -20, 2.0 ** -124, 2.0 ** -128, 2.0 ** -133]).repeat(10)[None, :, None, None]
    lens = torch.zeros(1, 1, dtype=I32)
    dk, dv, bt, new = check_append(x, -x, lens, None, 16, 64, seed=138)
    want = oracle_read(dk.cpu().numpy(), dv.cpu().numpy(), bt, new.cpu(), 60, lens)
    for g, w in zip(wgkv.kv4_read(dk, dv, bt.to(DEV), new, 60, dtype=dtype), want):
        assert torch.equal(g.cpu(), w.float().to(dtype))


def test_pools_of_one_buffer():
    """Pools side by side in one buffer are taken; the same pool for both, or
    pools that share a page, are refused before anything is written."""
    import wgkv
    from wgkv import _lib
    gen = torch.Generator().manual_seed(141)
    lens = torch.tensor([[5, 17]], dtype=I32)
    bt, n = table_for(lens + 9, 16, gen)
    k, v = rows(gen, 1, 9, 2, 64).to(DEV), rows(gen, 1, 9, 2, 64).to(DEV)
    both = torch.zeros(2 * n, 1, 640, dtype=torch.uint8, device=DEV)
    args = (bt.to(DEV), lens.to(DEV))
    for kc, vc in [(both[:n], both[:n]), (both[:n], both[n - 1:-1]), (both[n - 1:-1], both[:n])]:
        with pytest.raises(_lib.WGKVError):
            wgkv.kv4_append(k, v, kc, vc, *args)
    assert not both.any()
    apart = [torch.zeros(n, 1, 640, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for kc, vc in [(both[:n], both[n:]), apart]:
        wgkv.kv4_append(k, v, kc, vc, *args)
    assert torch.equal(both, torch.cat(apart))


def test_read_into_rows_of_any_layout():
    """Random layouts of a pair of outputs in one buffer, rows of both
    interleaved among others: filled where no two rows meet, else refused."""
    import wgkv
    from wgkv import _lib
    gen = torch.Generator().manual_seed(143)
    rng = np.random.default_rng(144)
    lens = torch.tensor([[3, 7], [5, 0], [1, 6]], dtype=I32)
    kc, vc, bt = random_cache(gen, lens, 16, 64)
    dk, dv, sl, tb = torch.from_numpy(kc).to(DEV), torch.from_numpy(vc).to(DEV), lens.to(DEV), bt.to(DEV)
    counts = [0, 0]
    for i in range(300):
        B, n, H = int(rng.integers(1, 4)), int(rng.integers(1, 6)), int(rng.integers(1, 3))
        sizes, strides, step = [2, B, n, H], [0] * 4, 64 + 8 * int(rng.integers(0, 2))
        for d in rng.permutation(4):  # nested, and in two of three cases one stride changed
            strides[d] = step
            step *= sizes[d]
        if i % 3:
            strides[int(rng.integers(0, 4))] = 8 * int(rng.integers(0, 8 * (i % 3) * B * n))
        at = np.add.outer(np.add.outer(np.arange(2) * strides[0], np.arange(B) * strides[1]),
                          np.add.outer(np.arange(n) * strides[2], np.arange(H) * strides[3])).ravel()
        meets = bool((np.diff(np.sort(at)) < 64).any())
        buf = torch.full((int(at.max()) + 64,), 7.0, dtype=torch.float16, device=DEV)
        out = tuple(torch.as_strided(buf, (B, n, H, 64), (*strides[1:], 1), j * strides[0]) for j in range(2))
        args = (dk, dv, tb[:B, :H], sl[:B, :H], n)
        counts[meets] += 1
        if meets:
            with pytest.raises(_lib.WGKVError):
                wgkv.kv4_read(*args, dtype=torch.float16, out=out)
            assert (buf == 7).all()
            continue
        wgkv.kv4_read(*args, dtype=torch.float16, out=out)
        want = wgkv.kv4_read(*args, dtype=torch.float16)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), (sizes, strides)
        assert int((buf == 7).sum()) >= buf.numel() - 64 * len(at)  # nothing between the rows is written
    assert min(counts) > 60, counts
