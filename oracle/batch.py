"""Packed-batch serving operators in 64 bits, straight from their definitions:
page tables one head after the other, attention one row after the other.  Test
infrastructure only."""
import numpy as np
import torch


def tables(lengths, cu, N, table, state, num_blocks, P, mask=None, free=()):
    """(lengths, slots, table, state, status) after a step; the arguments stay."""
    B, H, M = table.shape
    lens = [[min(max(int(x), 0), M * P) for x in row] for row in lengths]
    old = [row[:] for row in lens]
    out = table.copy()
    slots = np.full((N, H), -1, dtype=np.int64)
    nxt, held = max(int(state[0]), 0), min(max(int(state[1]), 0), len(free)) if len(free) else 0
    plan, need, over = [], 0, False
    for b in range(B):
        for h in range(H):
            rows = [n for n in range(cu[b], cu[b + 1]) if mask is None or mask[h, n]]
            new = -(-(lens[b][h] + len(rows)) // P) - -(-lens[b][h] // P)
            over |= lens[b][h] + len(rows) > M * P
            plan.append((b, h, rows, need, new))
            need += new
    take = min(need, held)
    after = [nxt, held if len(free) else int(state[1])]
    if over or nxt + need - take > num_blocks:
        return np.array(old), slots, out, np.array(after), 3
    ids = [int(x) for x in free[held - take:held]] + list(range(nxt, nxt + need - take))
    status = 0
    for b, h, rows, at, new in plan:
        p0 = -(-lens[b][h] // P)
        out[b, h, p0:p0 + new] = ids[at:at + new]
        for i, n in enumerate(rows):
            pos = lens[b][h] + i
            page = int(out[b, h, pos // P])
            if 0 <= page < num_blocks:
                slots[n, h] = page * P + pos % P
            else:
                status = 3
        lens[b][h] += len(rows)
    return np.array(lens), slots, out, np.array([after[0] + need - take, after[1] - take]), status


def attend(q, k, v, see, scale):
    """Rows q (R, D) over keys (T, D) where see (R, T): the output in 64 bits
    and how far a kernel may be from it.

    A kernel rounds each probability p to bf16 (a factor within 1 +- 2^-8) for
    the products with the values; the sum it divides by may hold the rounded or
    the unrounded ones.  The quotient is off by at most 2^-8 (sum p |v| + |o|
    sum p) / sum p, and the output's own rounding adds 2^-8 |o|.  Scores are
    fp32 sums of D products, off by at most (D + 2) 2^-24 sum |q k| |scale|,
    and their exponential's argument is rounded in fp32 (a few 2^-24 of its
    size), which act on every p as factors too."""
    q, k, v = q.double(), k.double(), v.double()
    R, D = q.shape
    out = torch.zeros(R, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if k.shape[0] == 0:
        return out, bound
    z = (q @ k.t().contiguous()) * scale
    z = torch.where(see, z, torch.full_like(z, float("-inf")))
    m = z.amax(1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    s = p.sum(1, keepdim=True)
    w = p / torch.where(s > 0, s, torch.ones_like(s))
    off = torch.where(see, (q.abs() @ k.abs().t().contiguous()) * abs(scale), torch.zeros_like(z)).amax(1, keepdim=True)
    rel = 2 * ((D + 2) * off + 8 * off + 8) * 2.0 ** -24 + 2.0 ** -8 * (1 + 2.0 ** -6)
    # a row takes no part in what it does not see, whatever stands there
    for i in range(0, R, 512):
        hide = ~see[i:i + 512]
        vi = v
        if not torch.isfinite(v).all():
            for r in range(i, min(R, i + 512)):
                vs = v[see[r]]
                out[r] = w[r, see[r]] @ vs
                bound[r] = rel[r] * (w[r, see[r]] @ vs.abs() + out[r].abs()) + out[r].abs() * 2.0 ** -8
            continue
        wi = w[i:i + 512].masked_fill(hide, 0)
        out[i:i + 512] = wi @ vi
        bound[i:i + 512] = rel[i:i + 512] * (wi @ vi.abs() + out[i:i + 512].abs()) + out[i:i + 512].abs() * 2.0 ** -8
    return out, bound + 1e-30


def prompt(q, k, v, cu, cuk, window, sinks, scale):
    """sink_window_attn: (output, bound), zeros for rows of no sequence."""
    N, Hq, D = q.shape
    H = k.shape[1]
    G = Hq // H
    out = torch.zeros(N, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(len(cu) - 1):
        nq, nk = cu[b + 1] - cu[b], cuk[b + 1] - cuk[b]
        p = torch.arange(nq, device=q.device)[:, None] + nk - nq
        j = torch.arange(nk, device=q.device)[None]
        see = (j <= p) & ((j > p - window) | (j < sinks))
        for h in range(Hq):
            o, e = attend(q[cu[b]:cu[b + 1], h], k[cuk[b]:cuk[b + 1], h // G], v[cuk[b]:cuk[b + 1], h // G], see, scale)
            out[cu[b]:cu[b + 1], h], bound[cu[b]:cu[b + 1], h] = o, e
    return out, bound


def rows_of(cache, table, n, P):
    """The first n tokens' rows of a head with this row of the page table."""
    t = torch.arange(n, device=cache.device)
    return cache.reshape(-1, cache.shape[2])[table.long()[t // P] * P + t % P]


def token(q, kc, vc, lens, table, scale, window=None, sinks=0, prefix=None):
    """One row per sequence: paged_decode_attn_window (window, sinks) or
    paged_decode_attn_shared (prefix = (lens, table, starts))."""
    B, _, Hq, D = q.shape
    H, P = lens.shape[1], kc.shape[1]
    G = Hq // H
    out = torch.zeros(B, 1, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(B):
        for h in range(H):
            n = int(lens[b, h])
            t = torch.arange(n, device=q.device)
            if window is not None:  # only visible tokens' pages hold anything
                t = t[(t >= n - window) | (t < sinks)]
            at = table[b, h].long()[t // P] * P + t % P
            k, v = kc.reshape(-1, D)[at], vc.reshape(-1, D)[at]
            if prefix is not None:
                plens, ptable, starts = prefix
                for g in range(plens.shape[0]):
                    if int(starts[g]) <= b < int(starts[g + 1]):
                        m = int(plens[g, h])
                        k = torch.cat([rows_of(kc, ptable[g, h], m, P), k])
                        v = torch.cat([rows_of(vc, ptable[g, h], m, P), v])
            see = torch.ones(G, k.shape[0], dtype=torch.bool, device=q.device)
            o, e = attend(q[b, 0, h * G:(h + 1) * G], k, v, see, scale)
            out[b, 0, h * G:(h + 1) * G], bound[b, 0, h * G:(h + 1) * G] = o, e
    return out, bound
