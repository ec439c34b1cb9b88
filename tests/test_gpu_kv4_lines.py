"""The 4-bit attention over lines cut into many ranges: tokens at every border
of a range, and around the page-id windows and offset corrections inside long
ranges, carry the softmax in turn (kv4_lines; what a lost one would change is
tested there on the CPU)."""
import numpy as np
import pytest
import torch

import kv4_lines as kl

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def cus():
    return torch.cuda.get_device_properties(DEV).multi_processor_count


def run_calls(line, most=None, run=None):
    import wgkv
    kc, vc, q, sl = (torch.as_tensor(x).to(DEV) for x in (line.kc, line.vc, line.q, line.lens))
    for i, (table, _) in enumerate(line.calls(most)):
        got = wgkv.paged_decode_attn_kv4(q, kc, vc, sl, table.to(DEV), line.scale)[:, 0].double().cpu().numpy()
        want, bound = line.expected(table, run)
        err = np.abs(got - want)
        assert (err <= bound).all(), (i, float((err / np.maximum(bound, 1e-30)).max()), np.argwhere(err > bound)[0])


@pytest.mark.parametrize("name", list(kl.BORDERS))
def test_attend_border_tokens(name):
    line = kl.Line(*kl.BORDERS[name], cus())
    print(f"[kv4 borders] {name}: {len(line.ranges)} ranges, {len(line.places)} places", flush=True)
    run_calls(line)


@pytest.mark.parametrize("per_wave,D,G,P", kl.LONG)
def test_attend_long_ranges(per_wave, D, G, P):
    line = kl.long_case(per_wave, D, G, P, cus())
    print(f"[kv4 long ranges] {per_wave} units a wave, D={D} G={G} P={P}, {sum(line.tokens)} tokens", flush=True)
    run_calls(line, most=20, run=per_wave * kl.UNIT)


def test_attend_corrects_the_offset():
    """134 million equal tokens, 65,536 of them a wave's (at 256 CUs)."""
    import wgkv
    case = kl.Flat
    D, P = case.D, case.P
    tile = np.zeros(10 * D, np.uint8)
    tile[:8 * D] = case.CODE * 17
    pairs = np.array([[case.STEP, case.MIDDLE]] * (D // 2), np.float32)
    tile[8 * D:] = torch.from_numpy(pairs).to(torch.bfloat16).view(torch.uint8).numpy().ravel()
    pages = 256
    cache = torch.from_numpy(np.tile(tile, (pages, P // 16, 1))).to(DEV)
    n = case.PER_WAVE * kl.UNIT * kl.waves_of(D, 8) * min(cus(), 512)
    table = (torch.arange(n // P, dtype=torch.int32, device=DEV) % pages).view(1, 1, -1)
    q = torch.zeros(1, 1, 8, D, dtype=torch.bfloat16, device=DEV)
    print(f"[kv4 offset] {n} tokens", flush=True)
    got = wgkv.paged_decode_attn_kv4(q, cache, cache, torch.full((1, 1), n, dtype=torch.int32, device=DEV), table, 0.125)
    assert float((got.double() - case.want()).abs().max()) <= case.bound()
