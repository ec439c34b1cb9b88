"""The 4-bit cache in 64 bits, on the CPU: quantisation, the tiles' bytes,
append, read and attention, written from the format's definition."""
import numpy as np
import torch

GROUP, TILE = 32, 16


def bf16(x):
    """float64 array -> the nearest bf16 values, float64 (through fp32)."""
    return torch.from_numpy(np.asarray(x, np.float64).astype(np.float32)).to(torch.bfloat16).double().numpy()


def bits16(x):
    """bf16 values held in float64 -> their 16 bits."""
    return torch.from_numpy(np.asarray(x, np.float64)).to(torch.bfloat16).view(torch.int16).numpy().astype(np.uint16)


def quantise(x):
    """x (..., D) float64 -> codes (..., D) int, s and m (..., D/32) float64."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    finite = np.isfinite(g).all(-1)
    with np.errstate(all="ignore"):
        gz = np.where(finite[..., None], g, 0.0)
        hi, lo = gz.max(-1), gz.min(-1)
        s, m = bf16((hi - lo) / 15.0), bf16((hi + lo) / 2.0)
        s = np.where(s < 2.0 ** -126, 0.0, s)
        bad = ~finite | ~np.isfinite(m)
        c = np.rint((gz - m[..., None]) / np.where(s == 0, 1.0, s)[..., None] + 7.5)  # ties to even
        c = np.clip(np.nan_to_num(c), 0, 15)
        c = np.where((s == 0)[..., None] | bad[..., None], 0, c).astype(np.int64)
    s, m = np.where(bad, np.nan, s), np.where(bad, np.nan, m)
    return c.reshape(x.shape), s, m


def values(c, s, m):
    g = c.reshape(*c.shape[:-1], c.shape[-1] // GROUP, GROUP)
    return (m[..., None] + s[..., None] * (g - 7.5)).reshape(c.shape)


def offsets(t, d, D, keys):
    """Byte of the code of (token t of a tile, d) and its shift."""
    if keys:
        word, nib = t * (D // 4) + d // 8 * 2 + d % 2, d % 8 // 2
    else:
        per = D // 16
        word = (((t // 4 * 16 + d // per) * 2 + t % 4 // 2) * (D // 64) + d % per // 4) * 2 + t % 2
        nib = d % 4
    return word * 2 + nib // 2, 4 * (nib % 2)


def scale_offset(t, g, D):
    """Byte of the (s, m) pair of group g of token t."""
    return 8 * D + ((t // 4 * (D // GROUP) + g) * 4 + t % 4) * 4


def put(tile, t, c, s, m, keys):
    """Writes token t's codes (D), s and m (D/32) into a tile (10*D bytes)."""
    D = c.shape[0]
    for d in range(D):
        at, sh = offsets(t, d, D, keys)
        tile[at] = (int(tile[at]) & ~(15 << sh)) | int(c[d]) << sh
    sb, mb = bits16(s), bits16(m)
    for g in range(D // GROUP):
        at = scale_offset(t, g, D)
        for j, w in ((0, sb[g]), (2, mb[g])):
            tile[at + j], tile[at + j + 1] = int(w) & 255, int(w) >> 8


def get(tile, t, D, keys):
    """Token t's codes, s and m."""
    d = np.arange(D)
    at, sh = offsets(t, d, D, keys)
    c = (tile[at].astype(np.int64) >> sh) & 15
    g = np.arange(D // GROUP)
    at = scale_offset(t, g, D)
    w = (tile[at].astype(np.uint32) | tile[at + 1].astype(np.uint32) << 8,
         tile[at + 2].astype(np.uint32) | tile[at + 3].astype(np.uint32) << 8)
    s, m = ((x << 16).view(np.float32).astype(np.float64) for x in w)
    return c, s, m


def append(k, v, kc, vc, table, lengths, mask=None):
    """Appends in place to kc/vc (num_blocks, P/16, 10*D) uint8 arrays; k/v
    (B, T, H, D) float64.  Returns (new lengths, whether anything was lost)."""
    B, T, H, D = k.shape
    P, n_pages, cap = kc.shape[1] * TILE, kc.shape[0], table.shape[2] * kc.shape[1] * TILE
    new, lost = lengths.copy(), False
    coded = [quantise(x) for x in (k, v)]
    for b in range(B):
        for h in range(H):
            p = min(max(int(lengths[b, h]), 0), cap)
            for t in range(T):
                if mask is not None and not mask[b, h, t]:
                    continue
                if p >= cap:
                    lost = True
                    break
                pg = int(table[b, h, p // P])
                if 0 <= pg < n_pages:
                    for cache, (c, s, m), keys in ((kc, coded[0], True), (vc, coded[1], False)):
                        put(cache[pg, p % P // TILE], p % TILE, c[b, t, h], s[b, t, h], m[b, t, h], keys)
                else:
                    lost = True
                p += 1
            new[b, h] = p
    return new, lost


def rows(cache, table_row, n, keys):
    """The first n tokens of a head: codes (n, D), s and m (n, D/32).  Page
    ids are clamped to the pool, as the attention does."""
    D, P = cache.shape[2] // 10, cache.shape[1] * TILE
    c, s, m = np.zeros((n, D), np.int64), np.zeros((n, D // GROUP)), np.zeros((n, D // GROUP))
    for p in range(n):
        pg = min(max(int(table_row[p // P]), 0), cache.shape[0] - 1)
        c[p], s[p], m[p] = get(cache[pg, p % P // TILE], p % TILE, D, keys)
    return c, s, m


WINDOW = 1024  # tokens a wave adds up before it takes the codes' offset out of its sums
PIECES = 272   # sums of waves (8) and workgroups (256) that are added up for a head, and a few more


def attend_head(x, kk, vv, scale, counts=None, run=None):
    """One query x (D) over a head's tokens, kk and vv their (codes, s, m):
    (out, bound), both (D).  A token may stand in the sequence ``counts``
    times.  The bound is how far a bf16 result may be off whose probabilities
    are rounded to bf16 for the product with the values (half a step, 2^-8, of
    p times what the code adds, s |c - 7.5|; the middles' part keeps fp32), with
    the scores' fp32 sums of D products of codes offset by up to 143, the final
    rounding (2^-8), and the fp32 sums over the tokens:
      * codes offset by up to 143 are added up over a window only, at most
        WINDOW tokens of one wave, before their offset goes (and the windows'
        errors are relative to the windows' own weights);
      * middles, windows without the offset and the weights, over the tokens
        that one wave takes (``run`` of them, all without it), then the pieces.
    An addition is off by 2^-24 of the sum so far, which is at most the whole;
    a token counts as one, though the matrix core adds 32 of them in a step,
    which leaves room for the sum that the offset is taken from."""
    D = x.shape[0]
    k, v = values(*kk), values(*vv)
    z = k @ x * scale
    w = np.ones(len(z)) if counts is None else np.asarray(counts, np.float64)
    n = w.sum()
    p = w * np.exp(z - z[w > 0].max(initial=-np.inf))
    p /= p.sum()
    o = p @ v
    steps, middles = np.repeat(vv[1], GROUP, 1), np.abs(np.repeat(vv[2], GROUP, 1))
    spread = steps * np.abs(vv[0] - 7.5)
    reach = np.repeat(kk[1], GROUP, 1) * 143 + np.abs(np.repeat(kk[2], GROUP, 1))
    dz = abs(scale) * (reach @ np.abs(x)) * (D + 8) * 2.0 ** -24 + (np.abs(z).max() + 8) * 2.0 ** -22
    sums = (min(n, WINDOW) + 8) * 143 * (p @ steps)
    if run is None:
        sums += (n + 8) * (p @ middles) + max(n - WINDOW, 0) * (p @ spread)
    else:
        sums += (run + PIECES) * (p @ middles + p @ spread + np.abs(o))
    return o, (2.0 ** -8 * np.abs(o) + 2.0 ** -8 * (p @ spread) * (1 + 2.0 ** -8)
               + 2 * (p * dz) @ np.abs(v) + 2 * (p @ dz) * np.abs(o) + 2.0 ** -24 * sums + 1e-30)


def attend(q, kc, vc, table, lengths, scale):
    """q (B, Hq, D) float64 -> (out, bound), both (B, Hq, D) float64: the
    attention, and how far a bf16 result may be from it (attend_head)."""
    B, Hq, D = q.shape
    H = table.shape[1]
    G = Hq // H
    out, bound = np.zeros((B, Hq, D)), np.zeros((B, Hq, D))
    cap = table.shape[2] * kc.shape[1] * TILE
    for b in range(B):
        for h in range(H):
            n = min(max(int(lengths[b, h]), 0), cap)
            if n == 0:
                continue
            kk, vv = rows(kc, table[b, h], n, True), rows(vc, table[b, h], n, False)
            for i in range(h * G, h * G + G):
                out[b, i], bound[b, i] = attend_head(q[b, i], kk, vv, scale)
    return out, bound


def pool_rows(kc, vc):
    """Every token of a pair of pools, in the pages' order."""
    N, P = kc.shape[0], kc.shape[1] * TILE
    return rows(kc, np.arange(N), N * P, True), rows(vc, np.arange(N), N * P, False)


def token_counts(table_row, n, pages, P):
    """How often each token of the pool stands among a head's first n."""
    counts = np.repeat(np.bincount(np.asarray(table_row[:n // P], np.int64), minlength=pages), P)
    if n % P:
        last = int(table_row[n // P]) * P
        counts[last:last + n % P] += 1
    return counts


def attend_shared(q, held, P, table, lengths, scale, run=None):
    """``attend`` for long sequences over few pages, which their tables name
    many times: each token of the pool (``held``: pool_rows) once, with its
    count in the head."""
    B, Hq, D = q.shape
    H = table.shape[1]
    G = Hq // H
    out, bound = np.zeros((B, Hq, D)), np.zeros((B, Hq, D))
    for b in range(B):
        for h in range(H):
            counts = token_counts(table[b, h], int(lengths[b, h]), len(held[0][0]) // P, P)
            live = counts > 0
            if not live.any():
                continue
            kk, vv = (tuple(y[live] for y in c) for c in held)
            for i in range(h * G, h * G + G):
                out[b, i], bound[b, i] = attend_head(q[b, i], kk, vv, scale, counts[live], run)
    return out, bound
