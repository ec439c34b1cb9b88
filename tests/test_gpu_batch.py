"""The packed-batch serving operators against the 64-bit oracle: tables, slots
and copied rows exactly, attention within the bound that its roundings give
(oracle.batch.attend)."""
import numpy as np
import pytest
import torch

from oracle import batch as ob

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
I32, BF16 = torch.int32, torch.bfloat16


def starts_of(lens, first=0):
    return [first + sum(lens[:i]) for i in range(len(lens) + 1)]


def i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def check_close(got, want, bound, what=""):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    worst = torch.where(torch.isnan(want), torch.zeros_like(want), (got - want).abs() - bound)
    assert worst.max().item() <= 0, f"{what}: {worst.max().item():.3e} over the bound"


# ---- page tables and rows ------------------------------------------------------
def check_tables(lens, req, H, P, mask=None, free=(), nxt=None, blocks=None, width=None, first=0, tail=0, held=None,
                 table=None, in_place=False, seed=0):
    """One step on the device and in the oracle.  lens (B, H) held tokens, req
    new ones per request; pages of held tokens come first in the pool."""
    import wgkv
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens)
    B = lens.shape[0]
    cu = starts_of(req, first)
    N = cu[-1] + tail
    pages = -(-lens // P)
    used = int(pages.sum())
    new = lens + (np.array(req)[:, None] if mask is None
                  else np.array([[int(mask[h, cu[b]:cu[b + 1]].sum()) for h in range(H)] for b in range(B)]))
    if table is None:
        width = width or int((-(-new // P)).max()) + 2
        table = np.full((B, H, width), -7, dtype=np.int32)
        perm = rng.permutation(used)
        at = 0
        for b in range(B):
            for h in range(H):
                n = min(int(pages[b, h]), width)
                table[b, h, :n] = perm[at:at + n]
                at += int(pages[b, h])
    if nxt is None:
        nxt = used + len(free)
    if blocks is None:
        blocks = nxt + int((-(-new // P) - pages).sum()) + 1
    state = [nxt, len(free) if held is None else held]
    want = ob.tables(lens, cu, N, table, state, blocks, P, mask, list(free))
    dt, dl, ds = i32(table), i32(lens), i32(state)
    status = torch.zeros(1, dtype=I32, device=DEV)
    kw = dict(out=dl, state_out=ds) if in_place else {}
    print(f"[tables] B={B} H={H} N={N} P={P} blocks={blocks} in_place={in_place}", flush=True)
    got = wgkv.build_block_tables(dl, i32(cu), N, dt, ds, blocks, P,
                                  g_mask=None if mask is None else torch.tensor(mask, device=DEV),
                                  free_ids=i32(list(free)) if len(free) else None, status=status, **kw)
    torch.cuda.synchronize()
    for x, y, name in zip((got[0], got[1], dt, got[2]), want, ("lengths", "slots", "table", "state")):
        assert np.array_equal(x.cpu().numpy(), y), f"{name}: {np.argwhere(x.cpu().numpy() != y)[:4]}"
    assert int(status) == want[4]
    if in_place:
        assert got[0] is dl and got[2] is ds
    else:
        assert np.array_equal(dl.cpu().numpy(), lens) and ds.tolist() == state
    return got


def held_tokens(rng, B, H, most):
    return rng.integers(0, most + 1, (B, H))


@pytest.mark.parametrize("B,H,P", [(1, 1, 16), (3, 2, 16), (64, 8, 16), (255, 8, 64), (256, 8, 16), (40, 17, 32), (7, 40, 16)])
@pytest.mark.parametrize("masked", [False, True])
def test_tables_of_a_decode_step(B, H, P, masked):
    rng = np.random.default_rng(B * H + P)
    lens = held_tokens(rng, B, H, 5 * P)
    mask = rng.random((H, B)) < 0.6 if masked else None
    check_tables(lens, [1] * B, H, P, mask, free=rng.permutation(1000)[:B // 2] + 10 ** 6, blocks=2 * 10 ** 6,
                 in_place=B % 2 == 0)


@pytest.mark.parametrize("req", [[256], [255, 1], [0, 0, 256], [1000], [256, 256], [257, 0, 511, 0, 0, 1], [3, 700, 64, 1],
                                 [5000, 1, 1, 1, 300]])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("H,P", [(1, 16), (3, 64), (18, 32)])
def test_tables_of_prompts(req, masked, H, P):
    rng = np.random.default_rng(sum(req) + H)
    lens = held_tokens(rng, len(req), H, 100)
    mask = rng.random((H, sum(req) + 9)) < rng.choice([0.02, 0.3, 0.98], (H, 1)) if masked else None
    for in_place in (False, True):
        check_tables(lens, req, H, P, mask, free=list(range(90000, 90013)), blocks=10 ** 5, first=4, tail=5,
                     in_place=in_place)


@pytest.mark.parametrize("masked", [False, True])
def test_tables_of_many_requests_in_a_tile(masked):
    """Hundreds of starts per tile of 256 tokens, empty requests among them, and
    more (request, head) pairs than one workgroup plans in LDS."""
    rng = np.random.default_rng(3)
    req = rng.choice([0, 1, 1, 2, 5], 900).tolist()
    mask = rng.random((8, sum(req))) < 0.5 if masked else None
    check_tables(held_tokens(rng, 900, 8, 40), req, 8, 16, mask)
    check_tables(held_tokens(rng, 900, 8, 40), req, 8, 16, mask, in_place=True)


@pytest.mark.parametrize("masked", [False, True])
def test_tables_of_many_heads(masked):
    """More (tile, head) pairs than a workgroup sums up in LDS."""
    rng = np.random.default_rng(4)
    mask = rng.random((1400, 300)) < 0.5 if masked else None
    check_tables(held_tokens(rng, 1, 1400, 40), [300], 1400, 16, mask)


def test_tables_without_tokens():
    check_tables([[0, 5], [16, 17]], [0, 0], 2, 16)
    check_tables([[0, 5], [16, 17]], [0, 0], 2, 16, first=3, tail=2)
    check_tables([[0]], [0], 1, 16, np.zeros((1, 0), bool))
    check_tables(np.zeros((300, 20), int), [0] * 300, 20, 16)
    check_tables(np.zeros((300, 20), int), [0] * 300, 20, 16, np.zeros((20, 0), bool))


@pytest.mark.parametrize("N", [40, 600])
@pytest.mark.parametrize("masked", [False, True])
def test_tables_refuse_what_does_not_fit(N, masked):
    mask = np.ones((2, 2 * N), bool) if masked else None
    lens = [[3, 0], [16, 31]]
    check_tables(lens, [N, N], 2, 16, mask, width=-(-N // 16))          # the fullest head would outgrow its table
    free = [70, 71, 72]
    need = sum(-(-(x + N) // 16) - -(-x // 16) for row in lens for x in row)
    check_tables(lens, [N, N], 2, 16, mask, free=free, nxt=100, blocks=100 + need - 4)  # one page short
    check_tables(lens, [N, N], 2, 16, mask, free=free, nxt=100, blocks=100 + need - 3)  # just enough
    check_tables(lens, [N, N], 2, 16, mask, free=free, held=2, nxt=100, blocks=100 + need - 3, in_place=True)
    check_tables(lens, [N, N], 2, 16, mask, free=free, held=99, nxt=100, blocks=10 ** 4)  # more than the list has


def test_tables_with_bad_pages():
    """A held page id outside the pool: its tokens get no slot and the status
    says so; so for ids of the free list."""
    table = np.full((1, 2, 4), 3, dtype=np.int32)
    table[0, 0, 0] = -1
    check_tables([[5, 5]], [30], 2, 16, table=table, nxt=10, blocks=50)
    check_tables([[5, 5]], [30], 2, 16, table=np.full((1, 2, 4), 3, dtype=np.int32), nxt=10, blocks=50, free=[7, 51, -2])


def test_tables_clamp_lengths_and_starts():
    """Lengths outside a table's range count as its ends; starts that do not
    ascend give some result within the buffers."""
    import wgkv
    check_tables([[-5, 100]], [0], 2, 16, width=3)
    for N in (100, 700):
        for mask in (None, torch.ones(2, N, dtype=torch.bool, device=DEV)):
            table = torch.full((3, 2, 8), -1, dtype=I32, device=DEV)
            guard = torch.full((4,), 5, dtype=I32, device=DEV)
            out, slots, _ = wgkv.build_block_tables(i32([[0, 3], [9, 0], [0, 0]]), i32([50, 10, N + 1000, -4]), N, table,
                                                    i32([0, 0]), 64, 16, g_mask=mask)
            torch.cuda.synchronize()
            assert guard.tolist() == [5] * 4 and int(slots.max()) < 64 * 16 and int(slots.min()) >= -1


def inside(shape, fill, margin=4096):
    """An int32 tensor with `margin` entries of `fill` before and behind it, and the whole."""
    n = int(np.prod(shape))
    whole = torch.full((n + 2 * margin,), fill, dtype=I32, device=DEV)
    return whole[margin:margin + n].view(shape), whole


@pytest.mark.parametrize("cu", [[50, 10, 1 << 30, -4], [700, 0, 700, 0], [-9, -9, -9, -9], [0, 650, 20, 640],
                                [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5], [300, 299, 298, 297]])
@pytest.mark.parametrize("N", [100, 256, 257, 700])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("H,in_place", [(2, False), (2, True), (1400, False)])
def test_tables_write_only_their_own_for_any_starts(cu, N, masked, H, in_place):
    """Starts that do not ascend or lie outside the tokens, lengths outside the
    table: what lies around the outputs stays, lengths and rows are in range."""
    import wgkv
    B, width, P, blocks = 3, 8, 16, 64
    table, t_all = inside((B, H, width), 77)
    out, o_all = inside((B, H), 77)
    slots, s_all = inside((N, H), 77)
    state, st_all = inside((2,), 77)
    free = i32(list(range(40, 50)))
    lens = torch.tensor([[0, 3], [9, -2 ** 31], [2 ** 31 - 1, 128]], dtype=I32, device=DEV).repeat(1, H // 2)
    state.copy_(i32([5, 10]))
    given = i32([5, 10])
    if in_place:
        out.copy_(lens)
        lens, given = out, state
    mask = (torch.arange(N * H, device=DEV).view(H, N) % 3 != 1) if masked else None
    print(f"[tables] cu={cu} N={N} H={H} masked={masked} in_place={in_place}", flush=True)
    wgkv.build_block_tables(lens, i32(cu), N, table, given, blocks, P, g_mask=mask, free_ids=free, out=out,
                            state_out=state, slots=slots)
    torch.cuda.synchronize()
    for whole, n in ((t_all, table.numel()), (o_all, out.numel()), (s_all, slots.numel()), (st_all, 2)):
        assert (whole[:4096] == 77).all() and (whole[4096 + n:] == 77).all()
    assert out.min() >= 0 and out.max() <= width * P
    assert slots.min() >= -1 and slots.max() < blocks * P


def test_tables_strides_and_buffers():
    import wgkv
    rng = np.random.default_rng(5)
    B, H, N, P = 3, 4, 300, 16
    big = torch.full((B, H + 2, 40), -1, dtype=I32, device=DEV)
    table = big[:, 1:-1]
    mask = torch.tensor(rng.random((N, H)) < 0.5, device=DEV).t()            # tokens not contiguous
    lens = torch.zeros(B, 2 * H, dtype=I32, device=DEV)[:, ::2]
    slots = torch.full((N, H), 9, dtype=I32, device=DEV)
    out = torch.full((B, H + 3), 77, dtype=I32, device=DEV)
    got = wgkv.build_block_tables(lens, i32([0, 100, 120, 300]), N, table, i32([5, 0]), 500, P,
                                  g_mask=mask.to(torch.uint8) * 7, out=out[:, :H], slots=slots)
    want = ob.tables(np.zeros((B, H), int), [0, 100, 120, 300], N, np.full((B, H, 40), -1, np.int32), [5, 0], 500, P,
                     mask.cpu().numpy())
    assert got[1] is slots and np.array_equal(slots.cpu().numpy(), want[1])
    assert np.array_equal(out[:, :H].cpu().numpy(), want[0]) and (out[:, H:] == 77).all()
    assert np.array_equal(table.cpu().numpy(), want[2]) and (big[:, 0] == -1).all() and (big[:, -1] == -1).all()


@pytest.mark.parametrize("N,H,D", [(1, 1, 64), (5, 3, 128), (300, 8, 64), (1000, 2, 40), (64, 2, 256)])
@pytest.mark.parametrize("layout", ["plain", "heads_first", "fused", "misaligned", "expanded"])
def test_append(N, H, D, layout):
    import wgkv
    gen = torch.Generator().manual_seed(N + D)
    P, blocks = 16, -(-N * H // 16) + 3
    k, v = (torch.randn(N, H, D, generator=gen).to(BF16).to(DEV) for _ in range(2))
    if layout == "heads_first":
        k = k.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "fused":
        qkv = torch.randn(N, 5 * H, D, generator=gen).to(BF16).to(DEV)
        k, v = qkv[:, 3 * H:4 * H], qkv[:, 4 * H:]
    elif layout == "misaligned":
        v = torch.cat([v.new_zeros(N, H, 3), v], 2)[..., 3:]
    elif layout == "expanded":
        v = v[:1].expand(N, H, D)
    slots = torch.randperm(blocks * P, generator=gen)[:N * H].view(N, H).to(I32)
    skip = torch.rand(N, H, generator=gen)
    slots = torch.where(skip < 0.1, torch.full_like(slots, -1), slots)
    slots = torch.where(skip > 0.95, torch.full_like(slots, blocks * P + 3), slots)
    kc, vc = (torch.full((blocks, P, D), 7.0, dtype=BF16, device=DEV) for _ in range(2))
    want = [c.clone().view(-1, D) for c in (kc, vc)]
    ok = (slots >= 0) & (slots < blocks * P)
    for w, x in zip(want, (k, v)):
        w[slots[ok].long().to(DEV)] = x[ok.to(DEV)]
    print(f"[append] N={N} H={H} D={D} {layout}", flush=True)
    wgkv.paged_append(k, v, kc, vc, slots.to(DEV))
    torch.cuda.synchronize()
    assert torch.equal(kc.view(-1, D), want[0]) and torch.equal(vc.view(-1, D), want[1])


@pytest.mark.parametrize("D", [40, 64, 128])
def test_append_of_tokens_with_one_slot(D):
    """Each 8 values of the row are one of the tokens'; other rows stay."""
    import wgkv
    N, H = 3000, 2
    k = torch.arange(N, device=DEV).to(torch.int16).view(BF16)[:, None, None].expand(N, H, D).contiguous()
    v = (torch.arange(N, device=DEV) + N).to(torch.int16).view(BF16)[:, None, None].expand(N, H, D).contiguous()
    kc, vc = (torch.full((4, 16, D), 7.0, dtype=BF16, device=DEV) for _ in range(2))
    slots = torch.full((N, H), -1, dtype=I32, device=DEV)
    slots[::3, 0] = 5
    slots[1::3, 1] = 40
    wgkv.paged_append(k, v, kc, vc, slots)
    torch.cuda.synchronize()
    for pool, base in ((kc, 0), (vc, N)):
        rows = pool.view(-1, D)
        bits = rows.view(torch.int16).long() - base
        for slot, first in ((5, 0), (40, 1)):
            pieces = bits[slot].view(-1, 8)
            assert (pieces == pieces[:, :1]).all() and (pieces % 3 == first).all()
            assert pieces.min() >= 0 and pieces.max() < N
        rest = torch.ones(64, dtype=torch.bool, device=DEV)
        rest[[5, 40]] = False
        assert (rows[rest] == 7).all()


# ---- prompts -------------------------------------------------------------------
def qkv(N, Nk, Hq, H, D, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(*s, generator=gen) for s in ((N, Hq, D), (Nk, H, D), (Nk, H, D)))
    return (q * spread).to(BF16).to(DEV), k.to(BF16).to(DEV), (v + 0.25).to(BF16).to(DEV)


def check_prompt(req, past, Hq, H, D, window, sinks, scale=None, first=0, tail=0, seed=0, spread=1.0):
    import wgkv
    cu = starts_of(req, first)
    cuk = cu if past is None else starts_of([a + b for a, b in zip(req, past)])
    N, Nk = cu[-1] + tail, cuk[-1] + (tail if past is None else 0)
    q, k, v = qkv(N, Nk, Hq, H, D, seed, spread)
    scale = D ** -0.5 if scale is None else scale
    print(f"[prompt] req={req[:8]} past={past and past[:8]} Hq={Hq} H={H} D={D} W={window} S={sinks}", flush=True)
    out = wgkv.sink_window_attn(q, k, v, i32(cu), window, sinks, scale, None if past is None else i32(cuk))
    torch.cuda.synchronize()
    want, bound = ob.prompt(q, k, v, cu, cuk, window, sinks, scale)
    check_close(out, want, bound)
    return out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 3), (64, 0), (100, 65), (1000, 4)])
def test_prompt_windows(D, G, window, sinks):
    check_prompt([300, 1, 65, 0, 129], None, 2 * G, 2, D, window, sinks, seed=G)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 200])
def test_prompt_lengths(n):
    check_prompt([n], None, 4, 1, 128, 40, 2, seed=n)
    check_prompt([n, 3], None, 4, 4, 64, 1 << 40, 0, seed=n, first=2, tail=3)


@pytest.mark.parametrize("past", [[0, 0, 0], [1, 63, 64], [500, 0, 777], [-3, -70, 5], [-64, 10, -1]])
@pytest.mark.parametrize("window,sinks", [(50, 5), (1, 1), (5000, 0), (128, 200)])
def test_prompt_behind_cached_keys(past, window, sinks):
    """The rows are the last of more keys, or there are fewer keys than rows
    (the first rows then see nothing)."""
    check_prompt([64, 70, 130], past, 8, 2, 128, window, sinks, seed=1)


@pytest.mark.parametrize("window,sinks", [(1 << 40, 0), ((1 << 31) - 1, (1 << 31) - 1), (3, 1 << 40)])
def test_prompt_largest_windows_with_fewer_keys_than_rows(window, sinks):
    check_prompt([64, 70, 130, 20], [-3, -70, 5, -10], 4, 2, 64, window, sinks, seed=1)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0, 1e-4])
def test_prompt_scales(scale):
    check_prompt([150, 20], None, 4, 2, 64, 33, 4, scale=scale)


def test_prompt_large_scores():
    """Scores far apart: the running maximum moves often."""
    check_prompt([400], None, 4, 1, 128, 150, 10, spread=30.0)


def test_prompt_long():
    check_prompt([5000, 3100], None, 8, 2, 128, 1024, 4)
    check_prompt([2500], [3000], 4, 1, 64, 1 << 30, 0)


@pytest.mark.parametrize("D,G,H", [(128, 4, 8), (64, 4, 8), (128, 3, 8), (64, 2, 16), (128, 8, 4)])
def test_prompt_more_items_than_workgroups(D, G, H):
    """A workgroup goes through several items, of odd and even numbers of tiles
    and (rows that see nothing) of none."""
    req, past = [900, 1, 130, 700, 300, 0, 1200, 64, 400], [0, 70, -129, 100, -300, 5, 64, 0, -200]
    check_prompt(req * 2, past * 2, G * H, H, D, 150, 3, seed=G)


def test_prompt_many_sequences():
    rng = np.random.default_rng(0)
    check_prompt(rng.choice([0, 1, 2, 3], 2048).tolist(), None, 2, 1, 64, 2, 1)


def test_prompt_starts_that_do_not_ascend():
    """They give some result, in the time of as many rows: not every stretch that
    they name over again, 64 million rows here."""
    import wgkv
    N, B = 64000, 2000
    q, k, v = qkv(N, N, 2, 1, 64, 3)
    cu = i32([0, N] * (B // 2) + [N])
    events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    times = []
    for starts in (i32([N * b // B for b in range(B + 1)]), cu):
        for _ in range(2):
            events[0].record()
            out = wgkv.sink_window_attn(q, k, v, starts, 1024, 4)
            events[1].record()
            torch.cuda.synchronize()
        times.append(events[0].elapsed_time(events[1]))
    assert out.shape == q.shape and times[1] < 20 * times[0] + 5
    for starts in ([50, 10, 30, -4], [2 ** 31 - 1, 0, -2 ** 31, 77], [90, 80, 70, 60], [0, 100, 0, 100]):
        for keys in (100, 5000):
            kk, vv = (t[:keys] for t in (k, v))
            ck = i32([0, keys // 3, keys // 2, keys])
            whole = torch.full((300, 2, 64), 7.0, dtype=BF16, device=DEV)
            wgkv.sink_window_attn(q[:100], kk, vv, i32(starts), 4000, 4, None, ck, out=whole[100:200])
            wgkv.sink_window_attn(q[:100], kk, vv, ck.clamp(max=100), 4000, 4, None, i32(starts), out=whole[100:200])
            torch.cuda.synchronize()
            assert (whole[:100] == 7).all() and (whole[200:] == 7).all()


def test_prompt_rows_of_no_sequence():
    import wgkv
    q, k, v = qkv(100, 100, 4, 2, 64, 0)
    cu = i32([20, 50, 90])
    got = wgkv.sink_window_attn(q, k, v, cu, 16, 2)
    assert not got[:20].any() and not got[90:].any() and got[20:90].abs().sum(2).min() > 0
    out = torch.full_like(q, 3.0)
    assert wgkv.sink_window_attn(q, k, v, cu, 16, 2, out=out) is out
    assert (out[:20] == 3).all() and (out[90:] == 3).all() and torch.equal(out[20:90], got[20:90])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_takes_nothing_from_what_it_does_not_see(bad, D):
    """Keys and values that are not finite in padding, behind the sequence and
    outside a row's window: rows that see them show it, others do not."""
    import wgkv
    req, first, tail, W, S = [200, 90], 5, 7, 40, 3
    cu = starts_of(req, first)
    q, k, v = qkv(cu[-1] + tail, cu[-1] + tail, 4, 2, D, 3)
    v[:first] = bad
    v[cu[-1]:] = bad
    k[:first] = bad
    k[cu[-1]:] = bad
    v[cu[0] + 70] = bad            # rows 70 .. 109 see it
    v[cu[1] + 89, 1, 5] = bad      # the last row's own
    out = wgkv.sink_window_attn(q, k, v, i32(cu), W, S)
    torch.cuda.synchronize()
    want, bound = ob.prompt(q, k, v, cu, cu, W, S, D ** -0.5)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), fine)
    assert not fine[cu[0] + 70:cu[0] + 110].any() and fine[cu[0] + 110:cu[1]].all() and fine[cu[0]:cu[0] + 70].all()
    check_close(torch.where(fine, out.double(), 0), torch.where(fine, want, 0), torch.where(fine, bound, 0))


@pytest.mark.parametrize("D,G,H", [(64, 1, 1), (64, 8, 3), (128, 4, 8), (128, 3, 2), (128, 2, 1)])
@pytest.mark.parametrize("req,past,window,sinks", [
    ([1], [9000], 1 << 30, 0), ([1], [9000], 4096, 64), ([5, 70, 0, 1], [4000, 0, 3, 700], 2000, 4),
    ([64, 33], [-20, 5000], 3000, 1), ([300], [2000], 2222, 100)])
def test_prompt_few_rows_behind_many_keys(D, G, H, req, past, window, sinks):
    """The keys of an item are cut into parts, some of which may be empty."""
    check_prompt(req, past, G * H, H, D, window, sinks, seed=G, first=2)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_parts_take_nothing_from_what_is_not_seen(bad, D):
    import wgkv
    cu, cuk, W, S = [0, 7, 47], [0, 3007, 6047], 1500, 3
    q, k, v = qkv(cu[-1], cuk[-1], 4, 2, D, 3)
    for t in (k, v):
        t[700:900] = bad           # before the windows
        t[3007 - 3] = bad          # the first sequence's rows 4 .. see it
    v[6047 - 1 - W - 20, 1, 9] = bad  # the second's rows .. 19, of KV head 1
    k[3007 + 1, 0] = bad           # a first token, of KV head 0: seen by all
    out = wgkv.sink_window_attn(q, k, v, i32(cu), W, S, None, i32(cuk))
    torch.cuda.synchronize()
    want, bound = ob.prompt(q, k, v, cu, cuk, W, S, D ** -0.5)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), fine) and fine[:4].all()
    check_close(torch.where(fine, out.double(), 0), torch.where(fine, want, 0), torch.where(fine, bound, 0))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D,G,H", [(64, 2, 2), (128, 4, 2), (128, 3, 1)])
@pytest.mark.parametrize("past", [[-20, 5000], [-20, 3], [-60, 4000], [-20, 0]])
def test_prompt_rows_that_see_nothing_give_zeros_whatever_the_values(bad, D, G, H, past):
    """More rows than keys: the first rows share their item's tiles with rows that
    see keys, and these hold values that are not finite.  With many keys behind
    the second sequence the call is cut into parts."""
    import wgkv
    req = [64, 33]
    cu, cuk = starts_of(req), starts_of([a + b for a, b in zip(req, past)])
    q, k, v = qkv(cu[-1], cuk[-1], G * H, H, D, 7)
    v[2] = bad                             # the first sequence's third key
    v[cuk[1] + 1, H - 1, 9] = bad          # one value, of the second's
    out = torch.full_like(q, 7.0)
    print(f"[prompt] past={past} G={G} H={H} D={D} bad={bad}", flush=True)
    wgkv.sink_window_attn(q, k, v, i32(cu), 3000, 1, None, i32(cuk), out=out)
    torch.cuda.synchronize()
    want, bound = ob.prompt(q, k, v, cu, cuk, 3000, 1, D ** -0.5)
    assert not out[:-past[0]].any(), "a row that sees nothing"
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), fine) and not fine[-past[0] + 2:64].any()
    check_close(torch.where(fine, out.double(), 0), torch.where(fine, want, 0), torch.where(fine, bound, 0))


def check_not_finite(out, want, bound):
    """NaN and infinities where the oracle has them, the rest within the bound."""
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out[torch.isinf(want)].double(), want[torch.isinf(want)]) and torch.isfinite(out[fine]).all()
    check_close(torch.where(fine, out.double(), 0), torch.where(fine, want, 0), torch.where(fine, bound, 0))


@pytest.mark.parametrize("D,G,H", [(64, 2, 1), (128, 4, 1), (128, 1, 2)])
@pytest.mark.parametrize("req,past", [([200], [0]), ([70, 40], [30, 2500])])
@pytest.mark.parametrize("window,sinks", [(40, 3), (65, 0), (3000, 0), (33, 100)])
@pytest.mark.parametrize("at", [(0,), (63,), (100,), (127, 5), (-1,), (-64, -65), (-100, 0, 50)])
def test_prompt_values_that_are_not_finite_anywhere(D, G, H, req, past, window, sinks, at):
    """Rows that see them show them and others do not, in calls cut along the keys
    or not."""
    import wgkv
    cu, cuk = starts_of(req), starts_of([a + b for a, b in zip(req, past)])
    q, k, v = qkv(cu[-1], cuk[-1], G * H, H, D, 11)
    for i, j in enumerate(at):
        v[j, 0, 9 * i + 1] = (float("inf"), float("nan"), -float("inf"))[i]
        v[j, H - 1, 40] = -float("inf") if i else float("inf")  # those of both signs: NaN
    print(f"[prompt] at={at} req={req} past={past} G={G} H={H} D={D} W={window} S={sinks}", flush=True)
    out = wgkv.sink_window_attn(q, k, v, i32(cu), window, sinks, None, i32(cuk))
    torch.cuda.synchronize()
    check_not_finite(out, *ob.prompt(q, k, v, cu, cuk, window, sinks, D ** -0.5))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("past", [0, 3000])
@pytest.mark.parametrize("bad", [False, True])
def test_prompt_values_next_to_the_largest(D, past, bad):
    """Scores that grow by 7 in log2 after the first tile, for 36 keys: 36 * 2^7 *
    2^120 passes fp32's range, under the row's own maximum the sums do not (36 +
    2500 * 2^-7 < 2^6 weights of values of 2^120).  `bad`: among them one that is
    not finite, which some rows see."""
    import wgkv
    N = 100
    q, k, v = qkv(N, N + past, 2, 1, D, 12)
    v = torch.sign(v.float()).mul(2.0 ** 120).to(BF16)
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    k[64 + past // 2:100 + past // 2, :, 0] = 7 * 0.6931 * D ** 0.5
    k[..., 1:] *= 0.01
    if bad:
        v[past + 50, 0, 3] = float("inf")
    cu, cuk = [0, N], [0, N + past]
    out = wgkv.sink_window_attn(q, k, v, i32(cu), 2500, 0, None, i32(cuk))
    torch.cuda.synchronize()
    want, bound = ob.prompt(q, k, v, cu, cuk, 2500, 0, D ** -0.5)
    assert torch.isfinite(want).all() == (not bad)
    check_not_finite(out, want, bound)


@pytest.mark.parametrize("past", [0, 3000])
def test_prompt_scores_of_minus_infinity(past):
    """Weights of 0: a finite value has no part, an infinite one makes NaN, and a
    row without other keys gives zeros."""
    import wgkv
    N, D = 100, 64
    q, k, v = qkv(N, N + past, 2, 1, D, 13)
    q[..., 0] = q[..., 0].abs() + 0.5
    k[past + 10:past + 20, :, 0] = -float("inf")
    v[past + 15, 0, 7] = float("inf")
    k[past + 60, 0, 0] = -float("inf")
    cu, cuk = [0, N], [0, N + past]
    scale = D ** -0.5
    for W in (3, 2000):
        out = wgkv.sink_window_attn(q, k, v, i32(cu), W, 0, None, i32(cuk))
        torch.cuda.synchronize()
        p, j = torch.arange(N, device=DEV)[:, None] + past, torch.arange(N + past, device=DEV)[None]
        see = (j <= p) & (j > p - W) & ~torch.isinf(k[:, 0, 0])[None]
        sees = (j <= p) & (j > p - W)
        for h in range(2):
            vv = v.clone()
            vv[past + 15, 0, 7] = 0
            want, bound = ob.attend(q[:, h], torch.nan_to_num(k[:, 0], neginf=0.0), vv[:, 0], see, scale)
            alone = see.sum(1) == 0
            assert not out[alone, h].any() and bool(alone.any()) == (W == 3)
            hit = torch.zeros_like(want, dtype=torch.bool)
            hit[:, 7] = sees[:, past + 15] & ~alone
            assert torch.equal(torch.isnan(out[:, h]), hit)
            check_close(torch.where(hit, 0, out[:, h].double()), torch.where(hit, 0, want), bound)


@pytest.mark.parametrize("D,what", [(128, "value"), (64, "row")])
def test_prompt_time_with_a_value_that_is_not_finite(D, what):
    """An infinite value of a first token, seen by every row, costs no row a pass
    of its own (4096 rows took more than 100 times as long)."""
    import wgkv
    q, k, v = qkv(4096, 4096, 8, 2, D, 14)
    cu = i32([0, 4096])
    events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]

    def best(n=5):
        times = []
        for _ in range(n):
            events[0].record()
            wgkv.sink_window_attn(q, k, v, cu, 1024, 4)
            events[1].record()
            torch.cuda.synchronize()
            times.append(events[0].elapsed_time(events[1]))
        return min(times)

    finite = best()
    v[1, 0, 3 if what == "value" else slice(None)] = float("inf")
    assert best() < 10 * finite


@pytest.mark.parametrize("past", [None, [150, 100]])
def test_prompt_rows_far_apart(past):
    """Keys more than 2^31 bytes apart, in one tile and over the call."""
    import wgkv
    req = [200, 100]
    cu = starts_of(req)
    cuk = cu if past is None else starts_of([a + b for a, b in zip(req, past)])
    Nk, stride = cuk[-1], 1 << 22
    q, k, v = qkv(cu[-1], Nk, 4, 2, 64, 5)
    big = torch.empty(Nk * stride, dtype=BF16, device=DEV)
    kf = big.as_strided((Nk, 2, 64), (stride, 64, 1), 0)
    vf = big.as_strided((Nk, 2, 64), (stride, 64, 1), 1024)
    kf.copy_(k)
    vf.copy_(v)
    out = wgkv.sink_window_attn(q, kf, vf, i32(cu), 70, 3, None, i32(cuk))
    want, bound = ob.prompt(q, k, v, cu, cuk, 70, 3, 64 ** -0.5)
    check_close(out, want, bound)
    assert torch.equal(out, wgkv.sink_window_attn(q, k, v, i32(cu), 70, 3, None, i32(cuk)))


@pytest.mark.parametrize("past", [None, [1500, 900]])
def test_prompt_values_that_are_not_finite_far_apart(past):
    """Keys more than 2^31 bytes apart: the last row of a block, and of a sequence,
    shows its own key's value."""
    import wgkv
    req = [100, 70]
    cu = starts_of(req)
    cuk = cu if past is None else starts_of([a + b for a, b in zip(req, past)])
    Nk, stride = cuk[-1], 1 << 21
    q, k, v = qkv(cu[-1], Nk, 4, 2, 64, 15)
    for i, j in enumerate((cuk[1] - 100, cuk[1] - 37, cuk[1] - 1, cuk[1] + 2, Nk - 7, Nk - 1)):
        v[j, i % 2, 5 * i] = (float("inf"), -float("inf"), float("nan"))[i % 3]
    big = torch.empty(Nk * stride, dtype=BF16, device=DEV)
    kf, vf = (big.as_strided((Nk, 2, 64), (stride, 64, 1), at) for at in (0, 1024))
    kf.copy_(k)
    vf.copy_(v)
    for window, sinks in ((70, 3), (2000, 0)):
        out = wgkv.sink_window_attn(q, kf, vf, i32(cu), window, sinks, None, i32(cuk))
        torch.cuda.synchronize()
        check_not_finite(out, *ob.prompt(q, k, v, cu, cuk, window, sinks, 64 ** -0.5))


def test_prompt_parts_captured():
    """Replays of a call that is cut into parts, with eager work between."""
    import wgkv
    q, k, v = qkv(40, 5040, 8, 2, 128, 1)
    cu, cuk = i32([0, 40]), i32([0, 5040])
    want = wgkv.sink_window_attn(q, k, v, cu, 4000, 4, None, cuk)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = wgkv.sink_window_attn(q, k, v, cu, 4000, 4, None, cuk)
    for i in range(4):
        out.fill_(-1)
        g.replay()
        other = wgkv.sink_window_attn(q + i, k, v, cu, 4000, 4, None, cuk)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert i == 0 or not torch.equal(other, want)


def test_prompt_layouts():
    import wgkv
    N, Hq, H, D = 150, 8, 2, 64
    q, k, v = qkv(N, N, Hq, H, D, 4)
    cu = i32([0, 60, 150])
    want = wgkv.sink_window_attn(q, k, v, cu, 30, 2)
    fused = torch.cat([q, k, v], 1)
    assert torch.equal(want, wgkv.sink_window_attn(fused[:, :Hq], fused[:, Hq:Hq + H], fused[:, Hq + H:], cu, 30, 2))
    t = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(want, wgkv.sink_window_attn(*t, cu, 30, 2))
    odd = [torch.cat([x.new_zeros(N, x.shape[1], 1), x], 2)[..., 1:] for x in (q, k, v)]
    assert torch.equal(want, wgkv.sink_window_attn(*odd, cu, 30, 2, out=torch.cat([q, q], 2)[..., 1:D + 1]))
    same = wgkv.sink_window_attn(q, k[:, :1].expand(N, H, D), v[:, :1].expand(N, H, D), cu, 30, 2)
    assert torch.equal(same[:, :4], want[:, :4])
    rows = torch.zeros(2 * N, Hq, D, dtype=BF16, device=DEV)
    wgkv.sink_window_attn(q, k, v, torch.stack([cu, cu], 1)[:, 0], 30, 2, out=rows[::2])
    assert torch.equal(rows[::2], want) and not rows[1::2].any()


# ---- one token per sequence ------------------------------------------------------
def paged(lens, P, D, seed, width=0, total=0, fill=None):
    """Page tables of heads with these token counts, -1 past the end, and pools."""
    gen = torch.Generator().manual_seed(seed)
    lens = torch.as_tensor(lens)
    pages = (lens + P - 1) // P
    width = max(width, int(pages.max()), 1)
    n = max(total, int(pages.sum()) + 2)
    perm = torch.randperm(n, generator=gen).to(I32)
    table = torch.full((*lens.shape, width), -1, dtype=I32)
    at = 0
    for i in np.ndindex(*lens.shape):
        c = int(pages[i])
        table[i][:c] = perm[at:at + c]
        at += c
    return table.to(DEV), perm[at:], n


def pools(n, P, D, seed):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, P, D, generator=gen) + x).to(BF16).to(DEV) for x in (0.0, 0.25)]


def query(B, Hq, D, seed, spread=1.0):
    return (torch.randn(B, 1, Hq, D, generator=torch.Generator().manual_seed(seed)) * spread).to(BF16).to(DEV)


def check_window(lens, Hq, P, D, window, sinks, scale=None, seed=0, spread=1.0):
    """Pages that no visible token lies in are given back: their entries are
    garbage, and unused pages of the pool hold NaN."""
    import wgkv
    lens = torch.as_tensor(lens)
    B, H = lens.shape
    table, spare, n = paged(lens, P, D, seed)
    kc, vc = pools(n, P, D, seed + 1)
    kc[spare.long()] = float("nan")
    vc[spare.long()] = float("nan")
    for b in range(B):
        for h in range(H):
            t = np.arange(int(lens[b, h]))
            seen = set((t[(t >= len(t) - window) | (t < sinks)] // P).tolist())
            for j in range(table.shape[2]):
                if j not in seen:
                    if j * P < len(t):
                        kc[int(table[b, h, j])] = float("nan")
                        vc[int(table[b, h, j])] = float("nan")
                    table[b, h, j] = int(spare[0])
    q = query(B, Hq, D, seed + 2, spread)
    scale = D ** -0.5 if scale is None else scale
    print(f"[window] lens={tuple(lens.shape)} Hq={Hq} P={P} D={D} W={window} S={sinks}", flush=True)
    out = wgkv.paged_decode_attn_window(q, kc, vc, lens.to(DEV, I32), table, window, sinks, scale)
    torch.cuda.synchronize()
    check_close(out, *ob.token(q, kc, vc, lens, table, scale, window, sinks))


@pytest.mark.parametrize("D,P", [(64, 16), (128, 16), (128, 64)])
@pytest.mark.parametrize("G", [1, 3, 4, 8])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (100, 4), (63, 40), (1 << 40, 0), (300, 1 << 40)])
def test_window(D, P, G, window, sinks):
    check_window([[0, 1, 15], [16, 17, 100], [333, 700, 1291]], 3 * G, P, D, window, sinks, seed=G)


@pytest.mark.parametrize("B,H", [(1, 1), (1, 8), (5, 8), (40, 2), (80, 3), (256, 8)])
def test_window_batches(B, H):
    rng = np.random.default_rng(B)
    check_window(rng.integers(0, 400, (B, H)), 2 * H, 16, 64, 70, 5)


def test_window_long_and_scales():
    check_window([[20000, 9000]], 8, 16, 128, 4096, 64)
    check_window([[90, 300]], 4, 16, 128, 50, 4, scale=-0.5)
    check_window([[90, 300]], 4, 16, 128, 50, 4, scale=0.0)
    check_window([[90, 3000]], 4, 16, 128, 2000, 4, spread=25.0)


def test_window_of_everything_is_the_whole_cache():
    import wgkv
    lens = torch.tensor([[100, 0], [257, 1000]])
    table, _, n = paged(lens, 16, 128, 3)
    kc, vc = pools(n, 16, 128, 4)
    q = query(2, 8, 128, 5)
    a = wgkv.paged_decode_attn_window(q, kc, vc, lens.to(DEV, I32), table, 5000, 0, 0.1)
    b = wgkv.paged_decode_attn(q, kc, vc, lens.to(DEV, I32), table, 0.1)
    assert torch.equal(a, b)


def test_window_masked_tokens_of_a_visible_page():
    """Tokens outside the window in a page that the window reaches into hold
    NaN: they have no part."""
    import wgkv
    lens = torch.tensor([[200, 150]])
    for D in (64, 128):
        table, _, n = paged(lens, 16, D, 3)
        kc, vc = pools(n, 16, D, 4)
        for h in range(2):
            for t in range(3, int(lens[0, h]) - 21):
                page = int(table[0, h, t // 16])
                kc[page, t % 16] = float("nan")
                vc[page, t % 16] = float("inf")
            for t in range(int(lens[0, h]), -(-int(lens[0, h]) // 16) * 16):  # behind the last token
                page = int(table[0, h, t // 16])
                kc[page, t % 16] = vc[page, t % 16] = float("nan")
        q = query(1, 4, D, 5)
        out = wgkv.paged_decode_attn_window(q, kc, vc, lens.to(DEV, I32), table, 21, 3, 0.1)
        check_close(out, *ob.token(q, kc, vc, lens, table, 0.1, 21, 3))


@pytest.mark.parametrize("B,H,G,D", [(1, 2, 4, 128), (5, 2, 1, 64), (2, 2, 5, 128), (33, 2, 4, 64)])
@pytest.mark.parametrize("window", [1, 70, 1 << 20])
@pytest.mark.parametrize("what", ["key nan", "key inf", "keys nan", "all keys nan", "query nan", "query inf", "value nan",
                                  "value inf"])
def test_window_shows_what_is_seen_and_not_finite(B, H, G, D, window, what):
    """In the results of the heads that see it, and of no others, however the
    call is cut (up to 64 heads of 4 query heads in chunks, others in ranges)."""
    import wgkv
    P, T = 16, 2100
    lens = torch.full((B, H), T)
    table, _, n = paged(lens, P, D, 3)
    kc, vc = pools(n, P, D, 4)
    q = query(B, G * H, D, 5)
    q[..., 0] = q[..., 0].abs() + 0.5      # (an infinite key's scores are +inf)
    kc[..., 0] = kc[..., 0].abs() + 0.5    # (and an infinite query's)
    b, h = B - 1, H - 1

    def rows(pool, t0, t1):
        return [pool[int(table[b, h, t // P]), t % P] for t in range(t0, t1)]

    kind, bad = what.rsplit(" ", 1)[0], float(what.rsplit(" ", 1)[1])
    if kind.startswith("query"):
        q[b, 0, h * G, 0] = bad
    elif kind == "keys":                   # the newest ones: every score of a wave's share
        for r in rows(kc, T - 64, T):
            r[:] = bad
    elif kind == "all keys":
        for r in rows(kc, 0, T):
            r[:] = bad
    else:
        rows(kc if kind == "key" else vc, T - 1, T)[0][0] = bad
    print(f"[window] B={B} H={H} G={G} D={D} W={window} {what}", flush=True)
    out = wgkv.paged_decode_attn_window(q, kc, vc, lens.to(DEV, I32), table, window, 0, 0.1)
    torch.cuda.synchronize()
    want, bound = ob.token(q, kc, vc, lens, table, 0.1, window, 0)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isinf(out), torch.isinf(want))
    hit = fine.new_zeros(fine.shape)
    mine = hit[b, 0, h * G:h * G + (1 if kind == "query" else G)]
    (mine[:, :1] if kind == "value" else mine)[:] = True
    assert torch.equal(~fine, hit)
    check_close(torch.where(fine, out.double(), 0), torch.where(fine, want, 0), torch.where(fine, bound, 0))


@pytest.mark.parametrize("B,H,G", [(1, 2, 4), (2, 2, 5)])
@pytest.mark.parametrize("T,window", [(3, 2), (2100, 70)])
def test_window_scores_of_minus_infinity_weigh_nothing(B, H, G, T, window):
    """A key whose score is -inf, and a head that sees no other."""
    import wgkv
    P, D = 16, 64
    lens = torch.full((B, H), T)
    table, _, n = paged(lens, P, D, 3)
    kc, vc = pools(n, P, D, 4)
    q = query(B, G * H, D, 5)
    q[..., 0] = q[..., 0].abs() + 0.5
    kc[int(table[0, 0, (T - 1) // P]), (T - 1) % P, 0] = -float("inf")
    for t in range(T - window, T):
        kc[int(table[0, 1, t // P]), t % P, 0] = -float("inf")
    out = wgkv.paged_decode_attn_window(q, kc, vc, lens.to(DEV, I32), table, window, 0, 0.1)
    torch.cuda.synchronize()
    assert not out[0, 0, G:2 * G].any()
    t = torch.arange(T - window, T - 1, device=DEV)
    at = table[0, 0].long()[t // P] * P + t % P
    see = torch.ones(G, len(t), dtype=torch.bool, device=DEV)
    want, bound = ob.attend(q[0, 0, :G], kc.view(-1, D)[at], vc.view(-1, D)[at], see, 0.1)
    check_close(out[0, 0, :G], want, bound)


def check_shared(lens, plens, starts, Hq, P, D, scale=None, seed=0, spread=1.0, given=None):
    import wgkv
    lens, plens = torch.as_tensor(lens), torch.as_tensor(plens)
    B, H = lens.shape
    need = int(((lens + P - 1) // P).sum())
    ptable, rest, n = paged(plens, P, D, seed, total=int(((plens + P - 1) // P).sum()) + need + 2)
    kc, vc = pools(n, P, D, seed + 1)
    table, left, _ = paged(lens, P, D, seed + 3)
    table = torch.where(table >= 0, rest.to(DEV)[table.clamp(min=0).long()], table)
    kc[rest[left.long()].long()] = float("nan")
    vc[rest[left.long()].long()] = float("nan")
    for ln, tb in ((lens, table), (plens, ptable)):  # rows behind the last token hold NaN
        for i in np.ndindex(*ln.shape):
            c = int(ln[i])
            if c % P:
                kc[int(tb[i][c // P]), c % P:] = float("nan")
                vc[int(tb[i][c // P]), c % P:] = float("nan")
    q = query(B, Hq, D, seed + 2, spread)
    scale = D ** -0.5 if scale is None else scale
    print(f"[shared] lens={tuple(lens.shape)} prefixes={tuple(plens.shape)} Hq={Hq} P={P} D={D}", flush=True)
    out = wgkv.paged_decode_attn_shared(q, kc, vc, lens.to(DEV, I32), table, plens.to(DEV, I32), ptable,
                                        i32(given or starts), scale)
    torch.cuda.synchronize()
    check_close(out, *ob.token(q, kc, vc, lens, table, scale, prefix=(plens, ptable, starts)))
    return out


@pytest.mark.parametrize("D,P", [(64, 16), (128, 16), (128, 64), (64, 32)])
@pytest.mark.parametrize("G", [1, 3, 4, 7, 8])
@pytest.mark.parametrize("B", [1, 3, 17])
def test_shared(D, P, G, B):
    rng = np.random.default_rng(B + G)
    check_shared(rng.integers(0, 90, (B, 2)), [[500, 37]], [0, B], 2 * G, P, D, seed=B)


@pytest.mark.parametrize("n", [0, 1, 15, 16, 31, 32, 33, 127, 128, 129, 1000])
def test_shared_lengths(n):
    check_shared([[n, 0], [0, n], [1, 5]], [[n, n // 2]], [0, 3], 4, 16, 128, seed=n)
    check_shared([[0, 0]] * 9, [[n, 3]], [0, 9], 16, 16, 64, seed=n)


@pytest.mark.parametrize("starts", [[0, 0, 5, 12], [2, 3, 3, 9], [0, 12, 12, 12], [4, 8, 10, 11]])
def test_shared_groups(starts):
    """Groups of one, none, all, and sequences of no group."""
    rng = np.random.default_rng(1)
    check_shared(rng.integers(0, 70, (12, 3)), rng.integers(0, 300, (3, 3)), starts, 12, 16, 128)


@pytest.mark.parametrize("B,H,N", [(64, 8, 1), (100, 2, 5), (256, 8, 2), (256, 8, 256), (40, 8, 1)])
def test_shared_batches(B, H, N):
    rng = np.random.default_rng(B)
    starts = [B * i // N for i in range(N + 1)]
    check_shared(rng.integers(0, 40, (B, H)), rng.integers(0, 200, (N, H)), starts, 4 * H, 16, 64)


def test_shared_long_and_scales():
    check_shared([[100, 3000]] * 20, [[20000, 7000]], [0, 20], 8, 16, 128)
    check_shared([[30, 40]] * 5, [[200, 100]], [0, 5], 8, 16, 128, scale=-0.4)
    check_shared([[30, 40]] * 5, [[200, 100]], [0, 5], 8, 16, 128, scale=0.0)
    check_shared([[30, 400]] * 12, [[2000, 100]], [0, 12], 8, 16, 128, spread=25.0)


def test_shared_nan_is_seen_by_those_who_see_it():
    import wgkv
    lens, plens = torch.tensor([[40, 9], [3, 50], [0, 0]]), torch.tensor([[64, 100]])
    table, _, n = paged(lens, 16, 128, 1)
    ptable, _, m = paged(plens, 16, 128, 2)
    ptable = torch.where(ptable >= 0, ptable + n, ptable)
    kc, vc = pools(n + m, 16, 128, 3)
    q = query(3, 4, 128, 4)
    vc[int(table[0, 0, 1]), 3, 7] = float("nan")    # value 7 of sequence 0's first head
    kc[int(table[1, 1, 2]), 0] = float("nan")       # a score of sequence 1's second head
    args = (lens.to(DEV, I32), table, plens.to(DEV, I32), ptable, i32([0, 3]))
    out = wgkv.paged_decode_attn_shared(q, kc, vc, *args, 0.1)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 0, :2, 7] = True
    bad[1, 0, 2:] = True
    assert torch.equal(torch.isnan(out), bad)
    kc[int(ptable[0, 0, 0]), 0] = float("nan")      # the prefix of every sequence's first head
    out = wgkv.paged_decode_attn_shared(q, kc, vc, *args, 0.1)
    assert torch.isnan(out[:, 0, :2]).all() and torch.isfinite(out[2, 0, 2:]).all()


@pytest.mark.parametrize("D", [64, 128])
def test_shared_more_chunks_than_workgroups(D):
    """A workgroup takes several chunks of prefixes besides its sequences."""
    rng = np.random.default_rng(D)
    B, H, N = 200, 8, 40
    check_shared(rng.integers(0, 200, (B, H)), rng.integers(0, 700, (N, H)), [B * i // N for i in range(N + 1)], 4 * H, 16,
                 D)


@pytest.mark.parametrize("N", [2, 64])
def test_shared_starts_that_do_not_ascend(N):
    """They are taken as the greatest so far: here all but the first prefix have
    no sequence, and nothing is written for them."""
    B, H = 96, 4
    starts = [0] + [B, 0] * (N // 2)
    rng = np.random.default_rng(N)
    lens, plens = rng.integers(0, 40, (B, H)), rng.integers(100, 300, (N, H))
    check_shared(lens, plens, [0] + [B] * N, 32, 16, 64, given=starts)


def test_shared_equals_one_table():
    """A prefix of whole pages and own pages, against the plain operator over
    the two tables behind each other."""
    import wgkv
    plens, lens = torch.tensor([[320, 320]]), torch.tensor([[5, 77], [0, 200], [64, 1]])
    table, _, n = paged(lens, 16, 128, 1)
    ptable, _, m = paged(plens, 16, 128, 2)
    ptable = torch.where(ptable >= 0, ptable + n, ptable)
    kc, vc = pools(n + m, 16, 128, 3)
    q = query(3, 8, 128, 4)
    a = wgkv.paged_decode_attn_shared(q, kc, vc, lens.to(DEV, I32), table, plens.to(DEV, I32), ptable, i32([0, 3]), 0.1)
    both = torch.cat([ptable.expand(3, 2, -1), table], 2).contiguous()
    b = wgkv.paged_decode_attn(q, kc, vc, (lens + 320).to(DEV, I32), both, 0.1)
    _, bound = ob.token(q, kc, vc, lens + 320, both, 0.1)
    check_close(a, b.double(), 2 * bound)


def test_token_operators_clamp_pages_and_lengths():
    """Page ids outside the pool and lengths outside the table stay within both."""
    import wgkv
    kc, vc = pools(6, 16, 64, 1)
    q = query(2, 4, 64, 2)
    table = i32([[[9, -5, 3], [0, 1, 2]], [[-1, 7, 100], [5, 5, 5]]])
    lens = i32([[1000, -4], [48, 20]])
    for out in (wgkv.paged_decode_attn_window(q, kc, vc, lens, table, 30, 2, 0.1),
                wgkv.paged_decode_attn_shared(q, kc, vc, lens, table, lens, table, i32([0, 1, 2]), 0.1),
                wgkv.paged_decode_attn_shared(q, kc, vc, lens, table, lens[:1], table[:1], i32([-3, 99]), 0.1),
                wgkv.paged_decode_attn_shared(q, kc, vc, lens, table, lens, table, i32([2, 0, 1]), 0.1)):
        torch.cuda.synchronize()
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("op", ["window", "shared"])
def test_token_layouts(op):
    import wgkv
    lens, plens = torch.tensor([[40, 9], [3, 150]]), torch.tensor([[64, 100]])
    table, _, n = paged(lens, 16, 64, 1)
    ptable, _, m = paged(plens, 16, 64, 2)
    ptable = torch.where(ptable >= 0, ptable + n, ptable)
    kc, vc = pools(n + m, 16, 64, 3)
    q = query(2, 4, 64, 4)
    lens, plens, starts = lens.to(DEV, I32), plens.to(DEV, I32), i32([0, 2])

    def call(q, lens, table, plens, ptable, starts, out=None):
        if op == "window":
            return wgkv.paged_decode_attn_window(q, kc, vc, lens, table, 33, 3, 0.1, out=out)
        return wgkv.paged_decode_attn_shared(q, kc, vc, lens, table, plens, ptable, starts, 0.1, out=out)

    want = call(q, lens, table, plens, ptable, starts)
    def strided(t, d):
        return torch.stack([t, t + 1], d).select(d, 0)
    assert torch.equal(want, call(q, strided(lens, 2), strided(table, 3), strided(plens, 2), strided(ptable, 3),
                                  strided(starts, 1)))
    assert torch.equal(want, call(q, strided(lens, 0), strided(table, 1), strided(plens, 0), strided(ptable, 0), starts))
    for qq in (q.transpose(2, 3).contiguous().transpose(2, 3), torch.cat([q[..., :1], q], 3)[..., 1:],
               torch.cat([q, q], 2)[:, :, :4]):
        assert torch.equal(want, call(qq, lens, table, plens, ptable, starts))
    buf = torch.full((2, 1, 4, 65), 5.0, dtype=BF16, device=DEV)
    assert torch.equal(want, call(q, lens, table, plens, ptable, starts, out=buf[..., 1:])) and (buf[..., 0] == 5).all()
    flip = torch.full((2, 1, 64, 4), 5.0, dtype=BF16, device=DEV).transpose(2, 3)
    assert call(q, lens, table, plens, ptable, starts, out=flip) is flip and torch.equal(want, flip)


# ---- together ----------------------------------------------------------------------
def test_a_batch_is_served():
    """Two prompts and their decode steps as they would be served: tables, rows
    and attention of the packed prompts, then steps of one token whose pages are
    built on the device, against a dense computation."""
    import wgkv
    Hq, H, D, P, W, S = 8, 2, 64, 16, 48, 4
    req, steps = [75, 130], 20
    cu = starts_of(req)
    blocks, width = 64, 12
    kc, vc = (torch.full((blocks, P, D), float("nan"), dtype=BF16, device=DEV) for _ in range(2))
    table = torch.full((2, H, width), -1, dtype=I32, device=DEV)
    lens, pages = torch.zeros(2, H, dtype=I32, device=DEV), i32([0, 0])
    status = torch.zeros(1, dtype=I32, device=DEV)
    q, k, v = qkv(sum(req) + 2 * steps, sum(req) + 2 * steps, Hq, H, D, 0)
    scale = D ** -0.5
    n = sum(req)
    got = wgkv.sink_window_attn(q[:n], k[:n], v[:n], i32(cu), W, S, scale)
    check_close(got, *ob.prompt(q[:n], k[:n], v[:n], cu, cu, W, S, scale))
    _, slots, _ = wgkv.build_block_tables(lens, i32(cu), n, table, pages, blocks, P, out=lens, state_out=pages,
                                          status=status)
    wgkv.paged_append(k[:n], v[:n], kc, vc, slots)
    rows = [list(range(cu[b], cu[b + 1])) for b in range(2)]
    one = i32([0, 1, 2])
    for i in range(steps):
        at = slice(n + 2 * i, n + 2 * i + 2)
        _, slots, _ = wgkv.build_block_tables(lens, one, 2, table, pages, blocks, P, out=lens, state_out=pages,
                                              status=status)
        wgkv.paged_append(k[at], v[at], kc, vc, slots)
        out = wgkv.paged_decode_attn_window(q[at].unsqueeze(1), kc, vc, lens, table, W, S, scale)
        for b in range(2):
            rows[b].append(n + 2 * i + b)
            see = torch.tensor([[t >= len(rows[b]) - W or t < S for t in range(len(rows[b]))]], device=DEV)
            for h in range(Hq):
                kk, vv = k[rows[b], h // 4], v[rows[b], h // 4]
                want, bound = ob.attend(q[n + 2 * i + b, h][None], kk, vv, see, scale)
                check_close(out[b, 0, h][None], want, bound)
    assert int(status) == 0 and lens.tolist() == [[95, 95], [150, 150]] and pages.tolist()[0] == 2 * (6 + 10)


def test_samples_of_one_prompt():
    """A gated prompt admitted once, then samples that share it: each sample's
    tokens go to its own pages, attention reads prefix and own pages."""
    import wgkv
    Hq, H, D, P, B, n = 8, 2, 128, 16, 6, 200
    blocks = 200
    kc, vc = (torch.full((blocks, P, D), float("nan"), dtype=BF16, device=DEV) for _ in range(2))
    q, k, v = qkv(n + 40 * B, n + 40 * B, Hq, H, D, 1)
    gate = torch.rand(H, n, generator=torch.Generator().manual_seed(2)).to(DEV) < 0.4
    ptable = torch.full((1, H, 20), -1, dtype=I32, device=DEV)
    pages = i32([0, 0])
    plens, slots, _ = wgkv.build_block_tables(torch.zeros(1, H, dtype=I32, device=DEV), i32([0, n]), n, ptable, pages,
                                              blocks, P, g_mask=gate, state_out=pages)
    wgkv.paged_append(k[:n], v[:n], kc, vc, slots)
    table = torch.full((B, H, 4), -1, dtype=I32, device=DEV)
    lens, cu = torch.zeros(B, H, dtype=I32, device=DEV), i32(range(B + 1))
    kept = [gate[h].nonzero().squeeze(1).tolist() for h in range(H)]
    mine = [[] for _ in range(B)]
    for i in range(20):
        at = slice(n + B * i, n + B * (i + 1))
        _, slots, _ = wgkv.build_block_tables(lens, cu, B, table, pages, blocks, P, out=lens, state_out=pages)
        wgkv.paged_append(k[at], v[at], kc, vc, slots)
        out = wgkv.paged_decode_attn_shared(q[at].unsqueeze(1), kc, vc, lens, table, plens, ptable, i32([0, B]), 0.1)
        for b in range(B):
            mine[b].append(n + B * i + b)
            for h in range(Hq):
                r = kept[h // 4] + mine[b]
                see = torch.ones(1, len(r), dtype=torch.bool, device=DEV)
                want, bound = ob.attend(q[n + B * i + b, h][None], k[r, h // 4], v[r, h // 4], see, 0.1)
                check_close(out[b, 0, h][None], want, bound)


def served_step(st):
    """A decode step in place: tables, rows, window attention, shared attention."""
    import wgkv
    wgkv.build_block_tables(st["lens"], st["one"], 3, st["table"], st["pages"], 90, 16, out=st["lens"],
                            state_out=st["pages"], slots=st["slots"], free_ids=st["free"])
    wgkv.paged_append(st["k"], st["v"], st["kc"], st["vc"], st["slots"])
    wgkv.paged_decode_attn_window(st["q"], st["kc"], st["vc"], st["lens"], st["table"], 20, 2, 0.1, out=st["w"])
    wgkv.paged_decode_attn_shared(st["q"], st["kc"], st["vc"], st["lens"], st["table"], st["plens"], st["ptable"],
                                  st["starts"], 0.1, out=st["s"])
    wgkv.sink_window_attn(st["pq"], st["k"], st["v"], st["one"], 20, 2, 0.1, out=st["p"])


def served_state(seed):
    gen = torch.Generator().manual_seed(seed)
    kc, vc = pools(90, 16, 64, seed)
    z = lambda *s: torch.zeros(*s, dtype=BF16, device=DEV)  # noqa: E731
    k, v = (torch.randn(3, 2, 64, generator=gen).to(BF16).to(DEV) for _ in range(2))
    q = query(3, 4, 64, seed)
    return {"lens": torch.zeros(3, 2, dtype=I32, device=DEV), "one": i32([0, 1, 2, 3]), "pages": i32([30, 3]),
            "free": i32([88, 85, 80]), "table": torch.zeros(3, 2, 6, dtype=I32, device=DEV),
            "slots": torch.zeros(3, 2, dtype=I32, device=DEV), "kc": kc, "vc": vc, "k": k, "v": v, "q": q,
            "plens": i32([[100, 30]]), "ptable": i32([[list(range(8)), list(range(10, 18))]]), "starts": i32([0, 3]),
            "w": z(3, 1, 4, 64), "s": z(3, 1, 4, 64), "p": z(3, 4, 64), "pq": q[:, 0].contiguous()}


def outputs(st):
    return [st[x].clone() for x in ("lens", "pages", "table", "slots", "kc", "vc", "w", "s", "p")]


def test_captured_steps_replay():
    """A captured step, replayed with eager work and waits between, gives the
    eager step's results every time; two graphs of one stream run on two."""
    eager, states = served_state(1), [served_state(1), served_state(1)]
    side = torch.cuda.Stream()
    served_step(served_state(2))  # the library and its scratch are there
    torch.cuda.synchronize()
    graphs = []
    with torch.cuda.stream(side):
        for st in states:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                served_step(st)
            graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(6):
        served_step(eager)
        want = outputs(eager)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        served_step(served_state(3 + i))
        torch.cuda.synchronize()
        for st in states:
            for x, y in zip(outputs(st), want):
                assert torch.equal(torch.nan_to_num(x.float()), torch.nan_to_num(y.float()))


def test_calls_on_two_streams():
    """Calls that overlap on two streams keep their scratch apart."""
    states = [served_state(11), served_state(12)]
    want = [served_state(11), served_state(12)]
    for st in want:
        for _ in range(8):
            served_step(st)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(8):
        for st, s in zip(states, streams):
            with torch.cuda.stream(s):
                served_step(st)
    torch.cuda.synchronize()
    for st, w in zip(states, want):
        for x, y in zip(outputs(st), outputs(w)):
            assert torch.equal(x, y)


def test_results_repeat():
    """The same call gives the same bits, whatever ran before."""
    import wgkv
    rng = np.random.default_rng(0)
    lens, plens = torch.tensor(rng.integers(0, 300, (30, 4))), torch.tensor(rng.integers(1000, 9000, (1, 4)))
    table, _, n = paged(lens, 16, 128, 1)
    ptable, _, m = paged(plens, 16, 128, 2)
    ptable = torch.where(ptable >= 0, ptable + n, ptable)
    kc, vc = pools(n + m, 16, 128, 3)
    q = query(30, 16, 128, 4)
    args = (q, kc, vc, lens.to(DEV, I32), table, plens.to(DEV, I32), ptable, i32([0, 30]), 0.09)
    first = wgkv.paged_decode_attn_shared(*args)
    for _ in range(5):
        check_shared([[3, 4]], [[50, 60]], [0, 1], 4, 16, 128)
        assert torch.equal(first, wgkv.paged_decode_attn_shared(*args))


def test_dispatcher_forms():
    import wgkv
    st = served_state(4)
    q, k, v, cu = st["pq"], st["k"], st["v"], st["one"]
    assert torch.equal(torch.ops.wgkv.sink_window_attn(q, k, v, cu, 20, 2), wgkv.sink_window_attn(q, k, v, cu, 20, 2))
    a = (st["q"], st["kc"], st["vc"], i32([[9, 20]] * 3), st["table"])
    assert torch.equal(torch.ops.wgkv.paged_decode_attn_window(*a, 5, 1, 0.1),
                       wgkv.paged_decode_attn_window(*a, 5, 1, 0.1))
    b = (st["plens"], st["ptable"], st["starts"], 0.1)
    assert torch.equal(torch.ops.wgkv.paged_decode_attn_shared(*a, *b), wgkv.paged_decode_attn_shared(*a, *b))
