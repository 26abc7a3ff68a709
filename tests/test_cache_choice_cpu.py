"""Frequencies between the ends of a ramp, and the kernel that attention over an 8-bit cache is given (no GPU needed)."""
import math

import pytest

import frisk_b200 as F
from frisk_b200 import capi


@pytest.mark.parametrize("scaling,low,high", [("wavelength", 1.0, 4.0), ("yarn", 1.0, 32.0)])
@pytest.mark.parametrize("dim,base,factor,trained", [(128, 10000.0, 16.0, 4096), (64, 500000.0, 8.0, 8192)])
def test_frequencies_between_the_ends(scaling, low, high, dim, base, factor, trained):
    """By the number of turns that a pair makes over the trained context, not by the pair's index."""
    got, _ = F.rotary_frequencies(dim, base, scaling=scaling, factor=factor, trained=trained, device="cpu")
    between = 0
    for i, g in enumerate(got.tolist()):
        f = base ** (-2 * i / dim)
        turns = trained * f / (2 * math.pi)
        stay = (turns - low) / (high - low)
        if 0 < stay < 1:
            between += 1
            assert math.isclose(g, f * stay + f / factor * (1 - stay), rel_tol=1e-13)
    assert between >= 3


@pytest.mark.parametrize("d,keys,batch,new,want", [(128, 4000, 8, 8, 16), (128, 4000, 8, 12, 16), (128, 4000, 8, 16, 128), (128, 1000, 8, 16, 16),
                                                   (128, 8000, 32, 8, 16), (128, 8000, 32, 12, 128), (64, 8000, 32, 8, 16), (64, 4000, 8, 24, 128)])
def test_the_choice_over_8_bit_caches(d, keys, batch, new, want):
    """What was measured to be the faster one (4 query heads a key head)."""
    width = -(-(keys + new) // 64)
    cache = capi.CacheDesc(4000, 64, 8, d, capi.E4M3, batch, width, width, batch * new)
    assert capi.cache_attention_tile_rows(cache, capi.CacheAttnDesc(32, capi.BF16, new, 0, 0, 0.1, 0)) == want
