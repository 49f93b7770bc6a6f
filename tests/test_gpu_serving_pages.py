"""Chunks over pages that hold no multiple of 8 tokens, whose tiles come by copies instead of TMA."""
import math

import pytest
import torch

from tests.test_gpu_serving import BF16, F16, attn_case, check_attn, run_attn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [BF16, F16])
@pytest.mark.parametrize("dim,bt", [(64, 12), (128, 5), (96, 20)])
def test_chunks_over_odd_pages_take_nothing_from_what_is_not_seen(cache, dim, bt):
    """Infinities and NaNs in V where some rows of a tile see a key and others do not: cleaned before the product and
    added to the rows that see them; in unused slots and pages they reach nothing.  Many items a CTA, and repeats."""
    lens = [(300, 260), (150, 100), (500, 70), (129, 129)]
    q, k, v, table, kl, starts = attn_case(6, lens, 4, 4, dim, bt, cache, cache)
    used = {p for r, (l, _) in enumerate(lens) for p in table[r][:-(-l // bt)]}
    for p in range(k.shape[0]):
        if p not in used:
            k[p], v[p] = math.nan, math.inf
    for r, (l, _) in enumerate(lens):
        if l % bt:
            k[table[r][l // bt], l % bt:], v[table[r][l // bt], l % bt:] = math.nan, math.nan
    base = (q, k, v, table, kl, starts)
    check_attn(base)
    clean, _ = run_attn(*base, 0.125)
    for pos, bad in ((30, math.inf), (100, -math.inf), (170, math.nan), (299, math.inf)):
        v2 = v.clone()
        v2[table[0][pos // bt], pos % bt, 1, 5] = bad
        first = max(pos - 40, 0)
        for _ in range(3):
            out, _ = run_attn(q, k, v2, table, kl, starts, 0.125)
            hit = out[first:260, 1, 5]
            assert (torch.isnan(hit) if math.isnan(bad) else hit == bad).all()
            out[first:260, 1, 5] = clean[first:260, 1, 5]
            assert torch.equal(out, clean)
