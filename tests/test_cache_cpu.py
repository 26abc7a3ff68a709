"""What the rotary and cache entries refuse before anything is launched, and the plain arithmetic around them (no GPU needed)."""
import ctypes
import math

import pytest
import torch

import frisk_b200 as F
from frisk_b200 import capi
from oracle import cache_oracle as co


def test_frequencies():
    f, a = F.rotary_frequencies(8, 100.0, device="cpu")
    assert a == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15, atol=0)
    assert torch.equal(F.rotary_frequencies(8, 100.0, scaling="linear", factor=4.0, device="cpu")[0], f / 4)
    n, _ = F.rotary_frequencies(8, 100.0, scaling="ntk", factor=4.0, device="cpu")
    assert n[0] == 1 and math.isclose(float(n[-1]), float(f[-1]) / 4, rel_tol=1e-14)
    y, a = F.rotary_frequencies(64, scaling="yarn", factor=16.0, trained=4096, device="cpu")
    plain, _ = F.rotary_frequencies(64, device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert math.isclose(a, 0.1 * math.log(16.0) + 1)
    assert torch.equal(y[turns > 32], plain[turns > 32]) and torch.equal(y[turns < 1], plain[turns < 1] / 16)
    w, a = F.rotary_frequencies(64, scaling="wavelength", factor=8.0, trained=8192, low=1.0, high=4.0, device="cpu")
    turns = 8192 * plain / (2 * math.pi)
    assert a == 1.0 and torch.equal(w[turns > 4], plain[turns > 4]) and torch.equal(w[turns < 1], plain[turns < 1] / 8)
    assert bool((w <= plain).all()) and bool((w >= plain / 8).all())
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, scaling="other"), dict(dim=8, scaling="yarn"), dict(dim=8, base=-1.0),
                dict(dim=8, scaling="linear", factor=0.5), dict(dim=8, scaling="yarn", trained=64, low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            F.rotary_frequencies(**bad, device="cpu")


def test_the_oracle_quantises_like_the_type():
    x = torch.randn(50, 64, dtype=torch.float64) * torch.logspace(-6, 6, 50, dtype=torch.float64)[:, None]
    x = x.float().double()
    codes, e = co.quantise(x)
    y = (x * torch.exp2(127 - e.double())[:, None]).float()
    assert float(y.abs().max()) <= 448 and bool((y.abs().amax(1) > 224).all())
    assert torch.equal(codes, y.to(torch.float8_e4m3fn).view(torch.uint8))
    assert torch.equal(co.values((codes, codes, e, e), 0), y.to(torch.float8_e4m3fn).double() * torch.exp2(e.double() - 127)[:, None])


def _cache_desc(**change):
    d = dict(pages=4, page=16, heads=2, D=64, dtype=capi.BF16, batch=1, table_width=4, table_stride=4, rows=3, k=1 << 20, v=2 << 20,
             k_exponent=None, v_exponent=None, table=3 << 20, starts=4 << 20, lengths=5 << 20)
    d.update(change)
    return capi.CacheDesc(**d)


def _attn(**change):
    d = dict(heads_q=4, dtype=capi.BF16, max_new=3, mask_width=0, mask_stride=0, scale=0.125, tile_rows=0)
    d.update(change)
    return capi.CacheAttnDesc(**d)


def test_descriptors_are_checked_on_the_host():
    """A size of zero says that the entry refuses the descriptor."""
    size = capi.cache_attention_workspace_bytes
    assert size(_cache_desc(), _attn()) > 0 and size(_cache_desc(dtype=capi.E4M3), _attn(dtype=capi.F16)) > 0
    for change in (dict(page=8), dict(page=24), dict(page=2048), dict(D=96), dict(D=256), dict(heads=0), dict(pages=0), dict(rows=-1), dict(batch=-1),
                   dict(batch=2, table_stride=3), dict(pages=1 << 40), dict(pages=1 << 62, heads=4), dict(table_width=(1 << 27) - 1, table_stride=1 << 27, page=16, heads=1, rows=1, batch=1),
                   dict(dtype=7), dict(dtype=capi.F32), dict(dtype=capi.F16),
                   dict(table_width=1 << 27, table_stride=1 << 27, heads=4096, rows=1 << 20, pages=1)):
        assert size(_cache_desc(**change), _attn()) == 0, change
    for change in (dict(heads_q=3), dict(heads_q=0), dict(heads_q=1 << 20), dict(dtype=capi.F32), dict(max_new=-1), dict(mask_width=-1),
                   dict(mask_stride=-1), dict(scale=math.nan), dict(scale=math.inf), dict(tile_rows=32), dict(tile_rows=-1)):
        assert size(_cache_desc(), _attn(**change)) == 0, change
        with pytest.raises(ValueError):
            capi.cache_attention_tile_rows(_cache_desc(), _attn(**change))


def test_the_choice_of_tiles():
    rows = capi.cache_attention_tile_rows
    long = dict(pages=4000, page=64, heads=8, D=128, batch=32, table_width=125, table_stride=125)
    for heads_q, new, want in ((8, 1, 16), (32, 4, 16), (32, 16, 128), (32, 32, 128), (32, 33, 256), (64, 64, 256)):
        assert rows(_cache_desc(**long), _attn(heads_q=heads_q, max_new=new)) == want
    # few key tiles: the cheaper beginning wins
    assert rows(_cache_desc(**dict(long, batch=1, table_width=8)), _attn(heads_q=32, max_new=16)) == 16
    assert rows(_cache_desc(**long), _attn(heads_q=32, max_new=16, tile_rows=256)) == 256
    # no hint: rows over sequences
    assert rows(_cache_desc(**dict(long, rows=32 * 16)), _attn(heads_q=32, max_new=0)) == 128


def test_null_contexts_are_refused():
    lib = capi.load()
    p, c, a, r = capi.Packed(1 << 20, 128, 64), _cache_desc(), _attn(), capi.RotaryDesc(1, 1, 0, 8, 8, capi.F32, 0, 0, 1, 1.0)
    assert lib.frisk_b200_rotary(None, r, 16, 16, p, None, p, None, None) == -7
    assert lib.frisk_b200_cache_write(None, c, capi.BF16, p, p, None) == -7
    assert lib.frisk_b200_cache_read(None, c, capi.BF16, p, p, None) == -7
    assert lib.frisk_b200_cache_attention(None, c, a, p, p, None, 16, 1 << 30, None) == -7
    assert ctypes.sizeof(capi.CacheDesc) == 8 + 16 + 8 + 16 + 7 * 8
    for code in (-10, -11, 3):
        assert "unknown" not in capi.strerror(code)


def test_what_is_not_on_a_device_is_refused():
    cache = F.paged_cache(4, 2, 16, 64, torch.float16, device="cpu")
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    for call in (lambda: F.cache_write(cache, x, x, i[None], i, i[:1]), lambda: F.cache_read(cache, i[None], i, i[:1], 1),
                 lambda: F.cache_attention(cache, x, i[None], i, i[:1]),
                 lambda: F.rotary(x, None, torch.zeros(1, dtype=torch.int64), F.rotary_frequencies(64, device="cpu")[0])):
        with pytest.raises(ValueError):
            call()
    for bad in (dict(page=8), dict(page=48), dict(d=80), dict(pages=0), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            F.paged_cache(**dict(dict(pages=2, heads=1, page=16, d=64, dtype=torch.float16, device="cpu"), **bad))
