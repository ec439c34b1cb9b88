"""Long lines of heads for the 4-bit attention's tests: the kernel's division
of work restated, and sequences over few shared pages in which a handful of
tokens at chosen places carry the softmax, so that each of them lost, doubled
or read from another page shows in the output."""
import numpy as np
import torch

from oracle import kv4 as ok

UNIT = 64      # tokens of a unit of work
FEWEST = 4     # units of a workgroup before more workgroups have none
WINDOW = 16    # units whose page ids a wave holds
PER_HEAD = 12  # tokens that carry a head's softmax
BACKGROUND = 8  # pages of tokens that carry nothing


def waves_of(D, G):
    """Waves of a workgroup."""
    return 4 if D == 128 and G > 4 else 8


def ranges(units, workgroups, waves):
    """The waves' ranges [first, end) of a line of so many units."""
    used = max(min(-(-units // FEWEST), workgroups), 1)
    out = []
    for w in range(used):
        first = w * (units // used) + min(w, units % used)
        n = units // used + (w < units % used)
        for i in range(waves):
            at = first + i * (n // waves) + min(i, n % waves)
            end = at + n // waves + (i < n % waves)
            if end > at:
                out.append((at, end))
    return out


def workgroups_of(tokens, P, width, cus):
    """Workgroups of a launch over heads with tables of this width."""
    units = -(-width * P // UNIT) * len(tokens)
    return min(-(-units // FEWEST), cus, 512)


def places(tokens, wave_ranges, offsets=None):
    """(head, token) at the borders of the waves' ranges within each head:
    first and last token of the first and last unit; with ``offsets`` those of
    the units so far from a range's (or, in it, the head's) begin instead."""
    units = [-(-t // UNIT) for t in tokens]
    starts = np.concatenate([[0], np.cumsum(units)])
    out = set()
    for first, end in wave_ranges:
        h = int(np.searchsorted(starts, first, side="right")) - 1
        while h < len(tokens) and starts[h] < end:
            lo, hi = max(first, starts[h]), min(end, starts[h + 1])
            if hi > lo:
                for u in ([lo, hi - 1] if offsets is None else [lo + o for o in offsets if lo + o < hi]):
                    t = int(u - starts[h]) * UNIT
                    out.add((h, t))
                    out.add((h, min(t + UNIT, tokens[h]) - 1))
            h += 1
    return sorted(out)


class Line:
    """Heads (B, H) of these lengths over a shared pool; ``calls`` deals the
    places out, at most PER_HEAD of a head and one of a page to a call."""

    def __init__(self, lens, D, G, P, cus, offsets=None, seed=0):
        self.lens, self.D, self.G, self.P = lens, D, G, P
        self.rng = np.random.default_rng(seed)
        B, H = lens.shape
        self.tokens = [int(n) for n in lens.flatten()]
        self.width = max(1, -(-max(self.tokens) // P))
        self.ranges = ranges(sum(-(-t // UNIT) for t in self.tokens),
                             workgroups_of(self.tokens, P, self.width, cus), waves_of(D, G))
        self.places = places(self.tokens, self.ranges, offsets)
        # a page per (place in a page, turn): all but that token background
        self.slots, pages = {}, BACKGROUND
        for i in sorted({t % P for _, t in self.places}):
            self.slots[i] = list(range(pages, pages + PER_HEAD))
            pages += PER_HEAD
        self.kc, self.vc = (self._pool(pages, keys) for keys in (True, False))
        self.held = ok.pool_rows(self.kc, self.vc)
        q = self.rng.normal(size=(B, H * G, D)) * 0.05
        q[..., :ok.GROUP] = 0.5  # group 0 of the keys tells the two kinds apart: by 32 in the score
        self.q = torch.from_numpy(q).to(torch.bfloat16)[:, None]
        self.scale = 1.0

    def _pool(self, pages, keys):
        D, P = self.D, self.P
        tiles = pages * P // ok.TILE
        out = self.rng.integers(0, 256, (tiles, 10 * D)).astype(np.uint8)
        s = self.rng.uniform(0.05, 0.25, (pages * P, D // ok.GROUP))
        m = self.rng.normal(size=s.shape) * (0.3 if keys else 1.0)
        if keys:
            s[:, 0], m[:, 0] = 2.0 ** -7, -1.0
            for i, turn in self.slots.items():
                m[np.array(turn) * P + i, 0] = 1.0
        pairs = torch.from_numpy(np.stack([s, m], -1)).to(torch.bfloat16).view(tiles, 4, 4, D // ok.GROUP, 2)
        out[:, 8 * D:] = pairs.transpose(2, 3).contiguous().view(torch.uint8).view(tiles, 2 * D).numpy()
        return out.reshape(pages, P // ok.TILE, 10 * D)

    def calls(self, most=None):
        """Tables (B, H, width) int32, and for each head the pool's tokens
        that carry it, until every place had its turn (or ``most`` calls)."""
        B, H = self.lens.shape
        left = [[] for _ in self.tokens]
        for h, t in self.places:
            left[h].append(t)
        for x in left:
            self.rng.shuffle(x)
        base = self.rng.integers(0, BACKGROUND, (len(self.tokens), self.width)).astype(np.int32)
        done = 0
        while any(left) and (most is None or done < most):
            table, carry = base.copy(), []
            for h, x in enumerate(left):
                turn, taken, later = {i: list(self.rng.permutation(v)) for i, v in self.slots.items()}, {}, []
                for t in x:
                    if len(taken) == PER_HEAD or t // self.P in taken:
                        later.append(t)
                    else:
                        taken[t // self.P] = (int(turn[t % self.P].pop()), t % self.P)
                for j, (page, _) in taken.items():
                    table[h, j] = page
                left[h] = later
                carry.append([page * self.P + i for page, i in taken.values()])
            done += 1
            yield torch.from_numpy(table).view(B, H, self.width), carry

    def expected(self, table, run=None):
        return ok.attend_shared(self.q[:, 0].double().numpy(), self.held, self.P, table.numpy(), self.lens.numpy(),
                                self.scale, run)


def uneven(extra):
    """Lines of a few units more than 256 workgroups' waves have ranges for."""
    units = 1024 + 3 * extra
    return torch.tensor([[units * 16 - 640, units * 16 + 640 - 63, 70, units * 32 - 100]], dtype=torch.int32)


def short_heads(B, H, seed, n=70):
    g = torch.Generator().manual_seed(seed)
    ln = torch.randint(0, n, (B, H), generator=g, dtype=torch.int32)
    ln[B - 1, H - 1], ln[0, 0], ln[0, H // 2] = 1500, 0, 2600
    return ln


# name: (lengths, D, G, P)
BORDERS = {
    **{f"uneven{e}": (uneven(e), 64, 2, 64) for e in (0, 1, 63, 65, 129, 500)},
    **{f"alone{n}": (torch.tensor([[n]], dtype=torch.int32), 64, 8, 16) for n in (65, 127, 257, 511, 513)},
    "alone4097": (torch.tensor([[4097]], dtype=torch.int32), 128, 4, 16),
    "pair3000": (torch.tensor([[3000, 17]], dtype=torch.int32), 128, 8, 16),
    "alone5003": (torch.tensor([[5003]], dtype=torch.int32), 64, 8, 32),
    "heads40": (short_heads(2, 20, 1, 900), 64, 2, 16),
    "heads90": (short_heads(3, 30, 2), 128, 4, 16),
    "heads300": (short_heads(5, 60, 3), 128, 8, 16),
}


def long_line(per_wave, D, G, workgroups, seed):
    """Heads of all lengths whose units are per_wave for every wave."""
    total = per_wave * waves_of(D, G) * workgroups
    rng = np.random.default_rng(seed)
    cut = np.sort(rng.choice(np.arange(200, total - 200), 5, replace=False))
    units = np.diff(np.concatenate([[0], cut, [total]]))
    units[[1, 4]] -= 2  # two short heads among them
    units = np.insert(units, [2, 4], [2, 2])
    lens = units * UNIT - rng.integers(0, UNIT, len(units))
    return torch.tensor(lens, dtype=torch.int32).view(2, -1)


LONG = [(per_wave, D, G, P) for per_wave in (16, 17, 32, 33) for D, G, P in ((64, 4, 64), (128, 4, 16), (128, 8, 16))]
LONG += [(33, 128, 6, 64), (49, 128, 1, 32)]
OFFSETS = (0, 1, 15, 16, 17, 31, 32, 33, 47, 48)


def long_case(per_wave, D, G, P, cus):
    line = Line(long_line(per_wave, D, G, min(cus, 512), per_wave + D + G), D, G, P, cus, OFFSETS, seed=per_wave)
    assert {e - f for f, e in line.ranges} == {per_wave}
    return line


class Flat:
    """One head of equal tokens under a query of zeros: every weight is 1, and
    what is left of the products with the values are their fp32 sums."""
    D, P, PER_WAVE, CODE = 64, 64, 1024, 15
    STEP, MIDDLE = 0.193359375, -1.4453125  # bf16 numbers; the step's significand is odd

    @classmethod
    def want(cls):
        return cls.MIDDLE + cls.STEP * (cls.CODE - 7.5)

    @classmethod
    def bound(cls):
        """Half a bf16 step of the output and the sums: a window's are exact
        (32 (128 + c) s has 16 bits, 32 of those 21; 135.5 n s is one rounding
        of a number below 2 * 143 s n); what is carried over, the output times
        the tokens so far, is rounded in each step of 32 tokens, together with
        the window's 143 s 1024 at most, and the middles' sum per token."""
        s, n = cls.STEP, cls.PER_WAVE * UNIT
        carried = (n / 32) * (n * abs(cls.want()) / 2 + 143 * s * ok.WINDOW)
        windows = (n / ok.WINDOW) * 2 * 143 * s * ok.WINDOW
        middles = (ok.WINDOW / 4) * abs(cls.MIDDLE) * n
        return 2.0 ** -8 * abs(cls.want()) + 2.0 ** -24 * ((carried + windows + middles) / n + ok.PIECES * abs(cls.want()) * 2)

    @classmethod
    def emulated(cls, flush):
        """A wave's sums in fp32, 32 tokens a step."""
        f = np.float32
        add, one = f(32 * (128 + cls.CODE) * cls.STEP), f(32 * cls.STEP)
        acc = total = corr = f(0)
        steps = cls.PER_WAVE * UNIT // 32
        for i in range(steps):
            acc, total, corr = f(acc + add), f(total + one), f(corr + f(32 * cls.MIDDLE))
            if (flush and i % 32 == 31) or i == steps - 1:
                acc = f(acc + f(-135.5 * float(total) + float(corr)))
                total = corr = f(0)
        return float(acc) / (32 * steps)
