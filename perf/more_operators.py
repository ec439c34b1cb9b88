"""Operators for serving a packed batch over paged per-head caches, as they are
measured: the page tables a step needs, the rows it writes, and attention with
a sliding window or over a prefix that sequences share.

Shapes are those of the repository's configurations (32 query heads, 8 KV
heads, head_dim 128, pages of 16, contexts up to 128K, about a fifth of the
tokens kept where a gate decides), with other groups, head dims, pages and odd
lengths beside them.

Kinds:
  tables  the pages, lengths and cache rows of a step's tokens
  append  the same, and the tokens' keys and values written to those rows
  prompt  attention of a packed batch of prompts, each row seeing the first
          tokens of its sequence and a window
  window  the same for one token per sequence over a paged cache
  shared  one token per sequence over a prefix that groups of sequences share
          and the sequences' own pages
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False  # True: run() calls the framework's kernels; False: the plain forms below


def listed():
    heads = {"Hq": 32, "Hkv": 8, "D": 128, "page": 16}
    kv = {"Hkv": 8, "D": 128, "page": 16}
    return [
        # a decode step of a large serving batch: one token per sequence, now and then a page
        {"name": "tables_b256_1", "kind": "tables", "B": 256, "T": 1, "held": 8000, "frac": 1.0, **kv},
        # eight ragged prompts whose gate keeps a fifth
        {"name": "tables_b8_gated", "kind": "tables", "B": 8, "T": 4096, "held": 0, "frac": 0.2, **kv},
        # a decode step of a few sequences of a model with small heads
        {"name": "append_b16_1_d64", "kind": "append", "B": 16, "T": 1, "held": 3001, "frac": 1.0, "Hkv": 4, "D": 64,
         "page": 64},
        # a 64K prompt in one piece, every token kept
        {"name": "append_64k_all", "kind": "append", "B": 1, "T": 65536, "held": 0, "frac": 1.0, **kv},
        # a handful of short chat prompts, small heads, an odd window
        {"name": "prompt_b7_600_d64", "kind": "prompt", "B": 7, "T": 601, "past": 0, "window": 127, "sinks": 4, "Hq": 16,
         "Hkv": 2, "D": 64},
        # chunks of four prompts behind what each has already cached, wide window
        {"name": "prompt_b4_chunk", "kind": "prompt", "B": 4, "T": 2048, "past": 6000, "window": 4096, "sinks": 64,
         "Hq": 32, "Hkv": 8, "D": 128},
        # a whole 32K prompt with the local window of the prefill configuration
        {"name": "prompt_32k", "kind": "prompt", "B": 1, "T": 32768, "past": 0, "window": 1024, "sinks": 4, "Hq": 32,
         "Hkv": 8, "D": 128},
        # one user's long chat, one token
        {"name": "window_b1_1k", "kind": "window", "B": 1, "ctx": 131072, "window": 1024, "sinks": 4, **heads},
        # a serving batch of long contexts, wide window
        {"name": "window_b64_4k", "kind": "window", "B": 64, "ctx": 16001, "window": 4096, "sinks": 64, **heads},
        # four samples of one short prompt
        {"name": "shared_b4_2k", "kind": "shared", "B": 4, "N": 1, "prefix": 2048, "kept": 1.0, "ctx": 100, **heads},
        # three system prompts, small heads, 8 query heads a KV head
        {"name": "shared_b60_8k_d64", "kind": "shared", "B": 60, "N": 3, "prefix": 8191, "kept": 1.0, "ctx": 2000,
         "Hq": 32, "Hkv": 4, "D": 64, "page": 32},
        # many requests on one long gated document
        {"name": "shared_b128_128k", "kind": "shared", "B": 128, "N": 1, "prefix": 131072, "kept": 0.3, "ctx": 600,
         **heads},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    Hkv = rng.choice([1, 2, 4, 8, 8])
    D = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 64])
    kind = rng.choice(["tables", "append", "prompt", "prompt", "window", "shared", "shared"])
    if kind in ("tables", "append"):
        T = rng.choice([1, _log_int(rng, 2, 30000)])
        B = _log_int(rng, 1, min(256, max(1, 60000 // T)))
        return {"kind": kind, "B": B, "T": T, "held": rng.choice([0, _log_int(rng, 1, 8000)]),
                "frac": rng.choice([1.0, round(rng.uniform(0.02, 0.6), 3)]), "Hkv": Hkv, "D": D, "page": page}
    G = rng.randint(1, 8)
    if kind == "prompt":
        B = _log_int(rng, 1, 12)
        G = min(G, 32 // Hkv)
        return {"kind": kind, "B": B, "T": _log_int(rng, 1, 8192 // B), "past": rng.choice([0, _log_int(rng, 1, 6000)]),
                "window": _log_int(rng, 1, 4096), "sinks": rng.choice([0, 1, 4, 64, 100]), "Hq": Hkv * G, "Hkv": Hkv,
                "D": D}
    if kind == "window":
        B = _log_int(rng, 1, 64)
        return {"kind": kind, "B": B, "ctx": _log_int(rng, 2, 131072), "window": _log_int(rng, 1, 4096),
                "sinks": rng.choice([0, 1, 4, 64]), "Hq": Hkv * min(G, 4), "Hkv": Hkv, "D": D, "page": page}
    B = _log_int(rng, 1, 128)
    return {"kind": kind, "B": B, "N": min(B, rng.choice([1, 1, 2, 5])),
            "prefix": _log_int(rng, 1, 32768), "kept": rng.choice([1.0, round(rng.uniform(0.1, 0.6), 3)]),
            "ctx": _log_int(rng, 1, 1000), "Hq": Hkv * min(G, 4), "Hkv": Hkv, "D": D, "page": page}


# ---- inputs -----------------------------------------------------------------
def _spread(n, lo, hi, seed):
    """n whole numbers spread evenly over [lo, hi], dealt in a random order
    (their total does not depend on the seed)."""
    out = [lo + round((hi - lo) * (i + 0.5) / n) for i in range(n)]
    random.Random(seed).shuffle(out)
    return out


def _request_lengths(c, seed):
    """New tokens of each sequence: ragged prompts, or one token each."""
    return _spread(c["B"], (c["T"] + 1) // 2 if c["B"] > 1 else c["T"], c["T"], seed)


def _past(c, seed):
    """Keys before each sequence's first row."""
    return _spread(c["B"], c["past"] // 3, c["past"], seed + 3)


def _held(c, seed):
    return _spread(c["B"] * c["Hkv"], c["held"] // 2, c["held"], seed + 1)


def _admitted(c, seed):
    """Tokens that the gate keeps, per (sequence, head)."""
    part = [round(c["frac"] * f * n) for n in _request_lengths(c, seed) for f in _spread(c["Hkv"], 50, 150, n)]
    return [min(a // 100, n) for a, n in zip(part, [n for n in _request_lengths(c, seed) for _ in range(c["Hkv"])])]


def _prefix_lens(c, seed):
    top = round(c["prefix"] * c["kept"])
    return _spread(c["N"] * c["Hkv"], top if c["kept"] >= 1.0 else top // 3, top, seed + 2)


def _own_lens(c, seed):
    """Cached tokens of each (sequence, head) of its own."""
    return _spread(c["B"] * c["Hkv"], c["ctx"] // 2, c["ctx"], seed)


def _group_starts(c):
    """N groups of sequences, of unlike sizes where there are several."""
    w = [2 + i % 3 for i in range(c["N"])]
    return [c["B"] * sum(w[:i]) // sum(w) for i in range(c["N"] + 1)]


def _pages_table(pages, first, width, gen, base, total):
    """int32 (heads, width): page ids of each head from column ``first`` on,
    ``pages`` of them, out of a random order of base .. base + total; -1
    elsewhere."""
    perm = torch.randperm(max(1, total), generator=gen, device="cuda").to(torch.int32) + base
    col = torch.arange(width, device="cuda")[None] - first[:, None]
    src = ((torch.cumsum(pages, 0) - pages)[:, None] + col).clamp(0, max(0, total - 1))
    inside = (col >= 0) & (col < pages[:, None])
    return torch.where(inside, perm[src], torch.full_like(src, -1, dtype=torch.int32))


def _states(shape, gen, keys):
    """Keys or values: N(0, 1), keys with a few channels of larger spread, as
    rotated keys of trained models have."""
    x = torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)
    if keys:
        x = x * torch.where(torch.arange(shape[-1], device="cuda") % 29 == 3, 3.0, 1.0)
    return x.to(torch.bfloat16)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    i32 = dict(dtype=torch.int32, device="cuda")
    B, H, D = c["B"], c["Hkv"], c["D"]
    st = {"kind": c["kind"], "c": c, "scale": D ** -0.5}
    if c["kind"] in ("tables", "append"):
        P = c["page"]
        req, held = _request_lengths(c, seed), _held(c, seed)
        N = sum(req)
        adm = _admitted(c, seed) if c["frac"] < 1.0 else [n for n in req for _ in range(H)]
        width = max((a + b + P - 1) // P for a, b in zip(held, adm)) + 3
        pages = torch.tensor([(n + P - 1) // P for n in held], device="cuda")
        used = int(pages.sum())
        free = used // 3 + 1  # pages that finished sequences gave back
        st["table"] = _pages_table(pages, torch.zeros_like(pages), max(1, width), gen, 0, used).view(B, H, -1)
        st["free"] = (torch.randperm(free, generator=gen, device="cuda").to(torch.int32) + used).contiguous()
        st["state"] = torch.tensor([used + free, free], **i32)
        st["blocks"] = used + free + sum((a + P - 1) // P + 1 for a in adm)
        st["lens"] = torch.tensor(held, **i32).view(B, H)
        st["cu"] = torch.tensor([sum(req[:i]) for i in range(B + 1)], **i32)
        st["N"] = N
        st["mask"] = None
        if c["frac"] < 1.0:  # exactly adm[b, h] tokens of every sequence and head, anywhere in it
            seq = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(req, device="cuda"))
            r = torch.rand(H, N, generator=gen, device="cuda", dtype=torch.float64) + seq[None]
            rank = r.argsort(1).argsort(1) - st["cu"].long()[seq][None]
            st["mask"] = rank < torch.tensor(adm, device="cuda").view(B, H).t()[:, seq]
        if c["kind"] == "append":
            st["k"], st["v"] = _states((N, H, D), gen, True), _states((N, H, D), gen, False)
            st["kc"] = torch.zeros(st["blocks"], P, D, dtype=torch.bfloat16, device="cuda")
            st["vc"] = torch.zeros_like(st["kc"])
        return st
    if c["kind"] == "prompt":
        req, past = _request_lengths(c, seed), _past(c, seed)
        keys = [a + b for a, b in zip(req, past)]
        st["cu"] = torch.tensor([sum(req[:i]) for i in range(B + 1)], **i32)
        st["cu_k"] = st["cu"] if c["past"] == 0 else torch.tensor([sum(keys[:i]) for i in range(B + 1)], **i32)
        st["most"], st["most_k"] = max(req), max(keys)
        st["q"] = torch.randn(sum(req), c["Hq"], D, generator=gen, device="cuda").to(torch.bfloat16)
        st["k"], st["v"] = _states((sum(keys), H, D), gen, True), _states((sum(keys), H, D), gen, False)
        return st
    P = c["page"]
    st["q"] = torch.randn(B, 1, c["Hq"], D, generator=gen, device="cuda").to(torch.bfloat16)
    lens = torch.tensor(_own_lens(c, seed), device="cuda")
    first = torch.zeros_like(lens)
    pages = (lens + P - 1) // P
    width = max(1, int(pages.max()))
    if c["kind"] == "window":  # pages behind the window were given back, but for the first tokens'
        sink = torch.minimum((torch.clamp(lens, max=c["sinks"]) + P - 1) // P, pages)
        first = torch.maximum(torch.clamp(lens - c["window"], min=0) // P, sink)
        own_pages = int((pages - first).sum())
        st["table"] = torch.where(torch.arange(width, device="cuda")[None] < sink[:, None],
                                  _pages_table(sink, torch.zeros_like(sink), width, gen, own_pages, int(sink.sum())),
                                  _pages_table(pages - first, first, width, gen, 0, own_pages)).view(B, H, width)
        total = own_pages + int(sink.sum())
    else:
        pl = torch.tensor(_prefix_lens(c, seed), device="cuda")
        pp = (pl + P - 1) // P
        st["plens"] = pl.to(torch.int32).view(c["N"], H)
        st["ptable"] = _pages_table(pp, torch.zeros_like(pp), max(1, int(pp.max())), gen, 0,
                                    int(pp.sum())).view(c["N"], H, -1)
        st["starts"] = torch.tensor(_group_starts(c), **i32)
        st["table"] = _pages_table(pages, first, width, gen, int(pp.sum()), int(pages.sum())).view(B, H, width)
        total = int(pp.sum()) + int(pages.sum())
    st["lens"] = lens.to(torch.int32).view(B, H)
    st["kc"], st["vc"] = _states((max(1, total), P, D), gen, True), _states((max(1, total), P, D), gen, False)
    return st


# ---- the plain forms ----------------------------------------------------------
def _plain_tables(st):
    """New lengths, cache rows, table and page state: head (b, h), in row-major
    order, takes the pages its new tokens need, the free list's last entries
    first (in list order), then the next unused pages."""
    c = st["c"]
    B, H, P, N = c["B"], c["Hkv"], c["page"], st["N"]
    dev = st["lens"].device
    mask = st["mask"] if st["mask"] is not None else torch.ones(H, N, dtype=torch.bool, device=dev)
    count = torch.zeros(H, N + 1, dtype=torch.int64, device=dev)
    count[:, 1:] = torch.cumsum(mask.to(torch.int64), 1)
    cu = st["cu"].long()
    at = count[:, cu]  # (H, B + 1)
    old = st["lens"].long()
    new = old + (at[:, 1:] - at[:, :-1]).t()
    p0, p1 = (old + P - 1) // P, (new + P - 1) // P
    need = (p1 - p0).reshape(-1)
    before = (torch.cumsum(need, 0) - need).view(B, H)
    nxt, held = st["state"][0].long(), st["state"][1].long()
    take = torch.minimum(need.sum(), held)
    col = torch.arange(st["table"].shape[2], device=dev)[None, None]
    i = before[..., None] + col - p0[..., None]  # the new page's number
    listed_id = st["free"].long()[(held - take + i).clamp(0, st["free"].numel() - 1)]
    ids = torch.where(i < take, listed_id, nxt + i - take)
    fresh = (col >= p0[..., None]) & (col < p1[..., None])
    st["table"].copy_(torch.where(fresh, ids, st["table"].long()).to(torch.int32))
    seq = torch.bucketize(torch.arange(N, device=dev), cu[1:], right=True)
    pos = old.t()[:, seq] + count[:, :-1] - at[:, seq]
    page = st["table"].long()[seq[None], torch.arange(H, device=dev)[:, None], pos // P]
    slots = torch.where(mask, page * P + pos % P, torch.full_like(pos, -1)).t().to(torch.int32).contiguous()
    state = torch.stack((nxt + need.sum() - take, held - take)).to(torch.int32)
    return new.to(torch.int32), slots, st["table"], state


def _plain_append(st):
    out = _plain_tables(st)
    keep = (out[1] >= 0).reshape(-1)
    rows = out[1].reshape(-1)[keep].long()
    for x, cache in ((st["k"], st["kc"]), (st["v"], st["vc"])):
        cache.view(-1, cache.shape[2])[rows] = x.reshape(-1, cache.shape[2])[keep]
    return (*out, st["kc"], st["vc"])


def _softmax_parts(z, valid):
    """exp(z - max) over the valid entries, and the max and sum."""
    z = torch.where(valid, z, torch.full_like(z, float("-inf")))
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    return p, m, p.sum(-1, keepdim=True)


def _join(parts):
    """(sum p v, max, sum p) of disjoint sets of keys -> the whole's output."""
    m = torch.stack([x[1] for x in parts]).amax(0)
    w = [torch.where(torch.isinf(x[1]), torch.zeros_like(m), torch.exp(x[1] - m)) for x in parts]
    s = sum(a * x[2] for a, x in zip(w, parts))
    return sum(a * x[0] for a, x in zip(w, parts)) / torch.where(s > 0, s, torch.ones_like(s))


def _attend(q, k, v, valid, scale):
    """(..., R, D) queries over (..., T, D) keys -> parts for _join."""
    p, m, s = _softmax_parts(torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale, valid)
    v = torch.where(valid.any(-2).unsqueeze(-1), v, torch.zeros_like(v))
    return torch.matmul(p, v), m, s


def _plain_prompt(st):
    """In a padded layout, tiles of 64 rows: the band of keys that the tile's
    windows reach, and the first tokens below each row's window."""
    c = st["c"]
    B, H, D, G, S = c["B"], c["Hkv"], c["D"], c["Hq"] // c["Hkv"], c["sinks"]
    W = min(c["window"], st["most_k"])
    dev, cq, ck = st["q"].device, st["cu"].long(), st["cu_k"].long()
    nq, nk = cq[1:] - cq[:-1], ck[1:] - ck[:-1]
    R = 64
    tiles = (st["most"] + R - 1) // R
    i = torch.arange(tiles * R, device=dev)[None]
    q = st["q"].float()[(cq[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)]
    q = q.view(B, tiles, R, H, G, D).permute(0, 1, 3, 4, 2, 5).reshape(B, tiles, H, G * R, D)
    pos = (i + (nk - nq)[:, None]).view(B, tiles, R)  # (B, tiles, R)
    j = pos[:, :, :1] - W + 1 + torch.arange(W + R - 1, device=dev)[None, None]  # (B, tiles, keys)
    at = (ck[:-1, None, None] + j).clamp(0, st["k"].shape[0] - 1)
    k = st["k"].float()[at].permute(0, 1, 3, 2, 4)
    v = st["v"].float()[at].permute(0, 1, 3, 2, 4)
    inside = (j >= 0) & (j < nk[:, None, None])
    see = inside[:, :, None] & (j[:, :, None] <= pos[..., None]) & (j[:, :, None] > pos[..., None] - W)
    see = see[:, :, None, None].expand(B, tiles, 1, G, R, W + R - 1).reshape(B, tiles, 1, G * R, W + R - 1)
    parts = [_attend(q, k, v, see, st["scale"])]
    if S:
        f = torch.arange(S, device=dev)[None]
        at = (ck[:-1, None] + f).clamp(0, st["k"].shape[0] - 1)
        k = st["k"].float()[at].permute(0, 2, 1, 3)[:, None]
        v = st["v"].float()[at].permute(0, 2, 1, 3)[:, None]
        see = (f < nk[:, None])[:, None, None] & (f[:, None, None] <= pos[..., None] - W)
        see = see[:, :, None, None].expand(B, tiles, 1, G, R, S).reshape(B, tiles, 1, G * R, S)
        parts.append(_attend(q, k, v, see, st["scale"]))
    o = _join(parts).view(B, tiles, H, G, R, D).permute(0, 1, 4, 2, 3, 5).reshape(B, tiles * R, H * G, D)
    return o[(i < nq[:, None])].to(torch.bfloat16)


def _rows(cache, table, pos, page):
    """fp32 rows of token positions (..., n) of each head's pages."""
    ids = torch.gather(table.long(), -1, (pos // page).clamp(0, table.shape[-1] - 1)).clamp(min=0)
    return cache.view(-1, cache.shape[2])[ids * page + pos % page].float()


def _plain_window(st):
    c = st["c"]
    B, H, D, G, P, S = c["B"], c["Hkv"], c["D"], c["Hq"] // c["Hkv"], c["page"], c["sinks"]
    W = min(c["window"], c["ctx"])
    lens = st["lens"].long()[..., None]
    j = torch.arange(S + W, device=lens.device).expand(B, H, -1)
    t = torch.where(j < S, j, lens - W + j - S)
    valid = torch.where(j < S, t < lens, (t >= S) & (t >= 0))
    t = t.clamp(min=0)
    q = st["q"].float().view(B, H, G, D)
    o = _join([_attend(q, _rows(st["kc"], st["table"], t, P), _rows(st["vc"], st["table"], t, P),
                       valid[:, :, None].expand(B, H, G, S + W), st["scale"])])
    return o.view(B, 1, H * G, D).to(torch.bfloat16)


def _plain_shared(st):
    """The prefix for each group's queries together, then each sequence's own
    tokens."""
    c = st["c"]
    B, H, D, G, P, N = c["B"], c["Hkv"], c["D"], c["Hq"] // c["Hkv"], c["page"], c["N"]
    q = st["q"].float().view(B, H, G, D)
    starts = st["starts"].long()
    group = torch.bucketize(torch.arange(B, device=q.device), starts[1:], right=True)
    place = torch.arange(B, device=q.device) - starts[group]
    most = max(b - a for a, b in zip(_group_starts(c)[:-1], _group_starts(c)[1:]))
    qg = torch.zeros(N, most, H, G, D, device=q.device)
    qg[group, place] = q
    qg = qg.permute(0, 2, 1, 3, 4).reshape(N, H, most * G, D)
    t = torch.arange(st["ptable"].shape[2] * P, device=q.device).expand(N, H, -1)
    valid = (t < st["plens"].long()[..., None])[:, :, None]
    parts = _attend(qg, _rows(st["kc"], st["ptable"], t, P), _rows(st["vc"], st["ptable"], t, P), valid, st["scale"])
    pre = [x.view(N, H, most, G, -1).permute(0, 2, 1, 3, 4)[group, place] for x in parts]
    t = torch.arange(st["table"].shape[2] * P, device=q.device).expand(B, H, -1)
    valid = (t < st["lens"].long()[..., None])[:, :, None]
    rest = _attend(q, _rows(st["kc"], st["table"], t, P), _rows(st["vc"], st["table"], t, P), valid, st["scale"])
    return _join([pre, rest]).view(B, 1, H * G, D).to(torch.bfloat16)


def _wgkv():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wg-kv_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import wgkv
    return wgkv


def run(state):
    st = state
    if not own:
        return {"tables": _plain_tables, "append": _plain_append, "prompt": _plain_prompt, "window": _plain_window,
                "shared": _plain_shared}[st["kind"]](st)
    wgkv, c = _wgkv(), st["c"]
    if st["kind"] in ("tables", "append"):
        lens, slots, pages = wgkv.build_block_tables(st["lens"], st["cu"], st["N"], st["table"], st["state"], st["blocks"],
                                                     c["page"], g_mask=st["mask"], free_ids=st["free"])
        if st["kind"] == "tables":
            return lens, slots, st["table"], pages
        wgkv.paged_append(st["k"], st["v"], st["kc"], st["vc"], slots)
        return lens, slots, st["table"], pages, st["kc"], st["vc"]
    if st["kind"] == "prompt":
        return wgkv.sink_window_attn(st["q"], st["k"], st["v"], st["cu"], c["window"], c["sinks"], st["scale"],
                                     cu_seqlens_k=st["cu_k"])
    if st["kind"] == "window":
        return wgkv.paged_decode_attn_window(st["q"], st["kc"], st["vc"], st["lens"], st["table"], c["window"],
                                             c["sinks"], st["scale"])
    return wgkv.paged_decode_attn_shared(st["q"], st["kc"], st["vc"], st["lens"], st["table"], st["plens"],
                                         st["ptable"], st["starts"], st["scale"])


def _pairs(c, seed):
    """(rows, visible keys) summed over a prompt batch's rows."""
    total = 0
    for n, past in zip(_request_lengths(c, seed), _past(c, seed)):
        p = np.arange(past, past + n, dtype=np.int64)
        total += int((np.minimum(p + 1, c["window"]) + np.clip(p + 1 - c["window"], 0, c["sinks"])).sum())
    return total


def work(case):
    c = case
    B, H, D = c["B"], c["Hkv"], c["D"]
    if c["kind"] in ("tables", "append"):
        N = sum(_request_lengths(c, 0))
        adm = sum(_admitted(c, 0)) if c["frac"] < 1.0 else N * H
        mask = N * H if c["frac"] < 1.0 else 0
        step = 8 * B * H + 4 * N * H + 8 * adm // c["page"] + mask + 4 * (B + 1)
        return {"bytes": step + (adm * D * 2 * 4 if c["kind"] == "append" else 0), "flops": 2 * N * H}
    Hq = c["Hq"]
    if c["kind"] == "prompt":
        rows, keys = sum(_request_lengths(c, 0)), sum(_request_lengths(c, 0)) + sum(_past(c, 0))
        return {"bytes": 4 * rows * Hq * D + 4 * keys * H * D, "flops": 4 * D * Hq * _pairs(c, 0)}
    if c["kind"] == "window":
        tokens = sum(min(n, c["window"] + c["sinks"]) for n in _own_lens(c, 0))
        return {"bytes": tokens * (4 * D + 4 / c["page"]) + 4 * B * Hq * D, "flops": 4 * D * Hq // H * tokens}
    pre, tokens = _prefix_lens(c, 0), sum(_own_lens(c, 0))
    size = [b - a for a, b in zip(_group_starts(c)[:-1], _group_starts(c)[1:])]
    seen = sum(size[i // H] * n for i, n in enumerate(pre)) + tokens
    return {"bytes": (sum(pre) + tokens) * (4 * D + 4 / c["page"]) + 4 * B * Hq * D, "flops": 4 * D * Hq // H * seen}


# ---- the definition in 64 bits ------------------------------------------------
def _exact_tables(st):
    """One head after the other, one page after the other."""
    c = st["c"]
    B, H, P = c["B"], c["Hkv"], c["page"]
    cu, lens, table = st["cu"].tolist(), st["lens"].tolist(), st["table"].cpu().numpy().copy()
    free, (nxt, held) = st["free"].tolist(), st["state"].tolist()
    mask = None if st["mask"] is None else st["mask"].cpu().numpy()
    slots = np.full((st["N"], H), -1, dtype=np.int64)
    plan, fresh = [], 0
    for b in range(B):
        for h in range(H):
            rows = np.arange(cu[b], cu[b + 1])
            if mask is not None:
                rows = rows[mask[h, cu[b]:cu[b + 1]]]
            new = -(-(lens[b][h] + len(rows)) // P) - -(-lens[b][h] // P)
            plan.append((b, h, rows, fresh, new))
            fresh += new
    take = min(fresh, held)
    ids = free[held - take:held] + list(range(nxt, nxt + fresh - take))
    for b, h, rows, at, new in plan:
        p0 = -(-lens[b][h] // P)
        table[b, h, p0:p0 + new] = ids[at:at + new]
        pos = lens[b][h] + np.arange(len(rows))
        slots[rows, h] = table[b, h, pos // P].astype(np.int64) * P + pos % P
        lens[b][h] += len(rows)
    return [torch.tensor(x) for x in (lens, slots, table, [nxt + fresh - take, held - take])]


def _exact_rows(q, k, v, scale):
    """(R, D) queries over (T, D) keys, all of them."""
    return torch.softmax(q.double() @ k.double().t() * scale, 1) @ v.double()


def exact(case, seed):
    c = case
    st = prepare(case, seed)
    H, D = c["Hkv"], c["D"]
    if c["kind"] in ("tables", "append"):
        lens, slots, table, state = _exact_tables(st)
        out = [x.to(torch.int32).cuda() for x in (lens, slots, table, state)]
        for cache, x in ((("kc", "k"), ("vc", "v")) if c["kind"] == "append" else ()):
            rows = torch.zeros(st[cache].numel() // D, D, dtype=torch.float64, device="cuda")
            n, h = torch.nonzero(out[1] >= 0, as_tuple=True)
            rows[out[1][n, h].long()] = st[x][n, h].double()
            out.append(rows.view(st[cache].shape))
        return tuple(out)
    G = c["Hq"] // H
    if c["kind"] == "prompt":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        cu, ck = st["cu"].tolist(), st["cu_k"].tolist()
        for b in range(c["B"]):
            nq, nk = cu[b + 1] - cu[b], ck[b + 1] - ck[b]
            for r0 in range(0, nq, 1024):
                r1 = min(nq, r0 + 1024)
                p = torch.arange(r0, r1, device="cuda")[:, None] + nk - nq
                lo = max(0, int(p[0]) - c["window"] + 1)
                j = torch.cat([torch.arange(min(c["sinks"], lo), device="cuda"),
                               torch.arange(lo, int(p[-1]) + 1, device="cuda")])
                hide = (j[None] > p) | ((j[None] <= p - c["window"]) & (j[None] >= c["sinks"]))
                for h in range(H):
                    k, v = st["k"][ck[b] + j, h].double(), st["v"][ck[b] + j, h].double()
                    q = st["q"][cu[b] + r0:cu[b] + r1, h * G:(h + 1) * G].double().transpose(0, 1)
                    z = torch.matmul(q, k.t().contiguous()) * st["scale"]
                    w = torch.softmax(z.masked_fill(hide[None], float("-inf")), 2)
                    out[cu[b] + r0:cu[b] + r1, h * G:(h + 1) * G] = torch.matmul(w, v).transpose(0, 1)
        return out
    P = c["page"]
    out = torch.zeros(c["B"], 1, c["Hq"], D, dtype=torch.float64, device="cuda")
    lens = st["lens"].tolist()
    kc, vc = st["kc"].view(-1, D), st["vc"].view(-1, D)
    for h in range(H):
        pre = {}
        for b in range(c["B"]):
            n = lens[b][h]
            t = torch.arange(n, device="cuda")
            if c["kind"] == "window":
                t = t[(t < c["sinks"]) | (t >= n - c["window"])]
            at = st["table"][b, h][t // P].long() * P + t % P
            if c["kind"] == "shared":
                g = next(i for i in range(c["N"]) if b < int(st["starts"][i + 1]))
                if g not in pre:
                    u = torch.arange(int(st["plens"][g, h]), device="cuda")
                    u = st["ptable"][g, h][u // P].long() * P + u % P
                    pre[g] = kc[u].double(), vc[u].double()
                k, v = torch.cat([pre[g][0], kc[at].double()]), torch.cat([pre[g][1], vc[at].double()])
            else:
                k, v = kc[at], vc[at]
            if k.shape[0]:
                out[b, 0, h * G:(h + 1) * G] = _exact_rows(st["q"][b, 0, h * G:(h + 1) * G], k, v, st["scale"])
    return out
