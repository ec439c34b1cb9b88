"""The long-line cases of the 4-bit attention's tests, on the CPU: that they
reach what they are for, and that a token lost or doubled would show."""
import numpy as np
import pytest

import kv4_lines as kl
from oracle import kv4 as ok

CUS = 256


def shows(line, table, carry, run=None):
    """Every carrying token left out, every one counted twice, and an output
    of zeros, exceed the bound of every query head."""
    B, H = line.lens.shape
    for bh, tokens in enumerate(carry):
        if not tokens:
            continue
        b, h = divmod(bh, H)
        counts = ok.token_counts(table[b, h].numpy(), line.tokens[bh], len(line.kc), line.P)
        live = np.flatnonzero(counts)
        kk, vv = (tuple(y[live] for y in c) for c in line.held)
        for i in {0, line.G - 1}:
            x = line.q[b, 0, h * line.G + i].double().numpy()
            o, bound = ok.attend_head(x, kk, vv, line.scale, counts[live], run)
            z = np.where(counts[live] > 0, ok.values(*kk) @ x * line.scale, -np.inf)
            w = counts[live] * np.exp(z - z.max())
            p, v = w / w.sum(), ok.values(*vv)
            at = np.searchsorted(live, tokens)
            assert p[at].sum() > 0.999 and (counts[tokens] == 1).all()
            assert (np.abs(o) > bound).any()
            for t in at:
                if len(tokens) > 1:  # a lone token's loss leaves the background
                    assert (np.abs((o - p[t] * v[t]) / (1 - p[t]) - o) > bound).any()
                    assert (np.abs((o + p[t] * v[t]) / (1 + p[t]) - o) > bound).any()


@pytest.mark.parametrize("name", list(kl.BORDERS))
def test_border_tokens_show(name):
    line = kl.Line(*kl.BORDERS[name], CUS)
    for table, carry in line.calls(most=2):
        shows(line, table, carry)


def test_every_place_has_its_turn():
    for name in ("uneven1", "heads90", "alone513"):
        line = kl.Line(*kl.BORDERS[name], CUS)
        seen = {}
        for table, carry in line.calls():
            t = table.view(-1, line.width)
            for h, tokens in enumerate(carry):
                for x in tokens:
                    page = np.flatnonzero(t[h].numpy() == x // line.P)
                    assert len(page) == 1
                    seen[(h, int(page[0]) * line.P + x % line.P)] = True
        assert sorted(seen) == line.places
    assert {(0, 0), (0, 63), (0, 64), (0, 512)} <= set(line.places)


@pytest.mark.parametrize("per_wave,D,G,P", kl.LONG)
def test_long_lines_reach_past_a_window(per_wave, D, G, P):
    """Waves of so many units, some within one head, some that begin inside
    one; the units around their 16th, 32nd and 48th have their turn."""
    line = kl.long_case(per_wave, D, G, P, CUS)
    assert len(line.ranges) == CUS * kl.waves_of(D, G)
    units = [-(-t // kl.UNIT) for t in line.tokens]
    starts = np.concatenate([[0], np.cumsum(units)])
    first, end = np.array(line.ranges).T
    head = np.searchsorted(starts, first, side="right") - 1
    inside = end <= starts[head + 1]
    assert inside.sum() > 900 and (~inside).sum() >= 4 and (inside & (first > starts[head])).sum() > 900
    offsets = {int(t // kl.UNIT + starts[h] - first[np.searchsorted(first, t // kl.UNIT + starts[h], side="right") - 1])
               for h, t in line.places}
    assert offsets >= {o for o in kl.OFFSETS if o < per_wave}
    for table, carry in line.calls(most=1):
        shows(line, table, carry, run=per_wave * kl.UNIT)


def test_sums_that_keep_the_offset_show():
    """What the corrections every 1024 tokens are for: the sum of codes offset
    by 128 over a wave's whole range, in fp32, is further off than the bound
    that the corrected one keeps (kv4_lines.Flat; the sums emulated)."""
    case = kl.Flat
    off, want, bound = case.emulated(flush=False), case.want(), case.bound()
    assert abs(off - want) > 4 * bound
    assert abs(case.emulated(flush=True) - want) <= bound
