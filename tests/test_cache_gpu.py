"""The paged cache and attention over it against 64 bits (oracle/cache_oracle.py, which derives the bounds)."""
import math

import pytest

from oracle import cache_oracle as co

pytestmark = pytest.mark.gpu


class Batch:
    """Ragged sequences over shuffled pages.  Pages that no sequence has, and page rows behind the keys, hold NaN."""

    def __init__(self, counts, lengths, hkv, group, d, page, dtype, held=None, seed=0, gap=0, fill=True, scales=(120, 134)):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.page = dtype, page
        held = dtype if held is None else held
        self.starts = [gap]
        for n in counts:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1] + gap
        need = [-(-(n + m) // page) for n, m in zip(counts, lengths)]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g)
        table = torch.full((len(counts), max(need + [0]) + 1), -7, dtype=torch.int32)  # (entries behind the last page are never read)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n].int()
            at += n
        shape = pages, hkv, page, d
        cache = [torch.full(shape, math.nan, dtype=torch.float32) for _ in range(2)]
        exps = [torch.full(shape[:3], 255, dtype=torch.uint8) for _ in range(2)]
        for b in range(len(counts) if fill else 0):
            j = torch.arange(lengths[b] + counts[b])
            for i in range(2):
                where = (table[b].long()[j // page], slice(None), j % page)
                cache[i][where] = torch.randn(len(j), hkv, d, generator=g)
                exps[i][where] = torch.randint(*scales, (len(j), hkv), generator=g, dtype=torch.uint8)
        if held == torch.float8_e4m3fn:
            cache = [torch.where(torch.isnan(c), c, (c * 100).clamp(-448, 448)).to(held) for c in cache] + exps
            if not fill:
                cache = [torch.full(shape, 0x55, dtype=torch.uint8).view(held) for _ in range(2)] + exps
        else:
            cache = [c.to(dtype) for c in cache]
        self.cpu = tuple(cache)
        self.table_cpu = table
        # queries, keys and values as columns of one buffer
        h = hkv * group
        self.buf = torch.randn(self.rows, (h + 2 * hkv) * d, generator=g).to(dtype)
        dev = self.buf.cuda()
        self.q = dev[:, :h * d].view(self.rows, h, d)
        self.k = dev[:, h * d:(h + hkv) * d].view(self.rows, hkv, d)
        self.v = dev[:, (h + hkv) * d:].view(self.rows, hkv, d)
        self.lengths = list(lengths)
        self.refresh()
        self.plan = (table.cuda(), torch.tensor(self.starts, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
        self.host = (table, self.starts, self.lengths)

    def refresh(self):
        self.cache = tuple(t.cuda() for t in self.cpu)

    def tile_rows(self, max_new):
        from frisk_b200 import capi
        code = {"float16": capi.F16, "bfloat16": capi.BF16, "float8_e4m3fn": capi.E4M3}
        (pages, heads, page, d), h = self.cpu[0].shape, self.q.shape[1]
        cache = capi.CacheDesc(pages, page, heads, d, code[str(self.cpu[0].dtype)[6:]], len(self.lengths), self.plan[0].shape[1],
                               self.plan[0].stride(0), self.rows)
        return capi.cache_attention_tile_rows(cache, capi.CacheAttnDesc(h, code[str(self.dtype)[6:]], max_new, 0, 0, 1.0, 0))

    def inside(self):
        import torch
        i = torch.zeros(self.rows, dtype=torch.bool)
        i[self.starts[0]:self.starts[-1]] = True
        return i


def bits(t):
    import torch
    return t.detach().cpu().contiguous().view(torch.uint8)


def same(a, b):
    import torch
    return all(torch.equal(bits(x), bits(y)) for x, y in zip(a, b))


def tree(batch, seed, kind="tree", width=None):
    import torch
    g = torch.Generator().manual_seed(seed)
    counts = [b - a for a, b in zip(batch.starts[:-1], batch.starts[1:])]
    width = max(counts) if width is None else width
    mask = torch.zeros(batch.rows, width, dtype=torch.bool)
    for first, n in zip(batch.starts[:-1], counts):
        if kind == "random":  # rows may be empty, rows may look ahead
            mask[first:first + n] = torch.rand(n, width, generator=g) < 0.3
            continue
        for i in range(n):
            if i:
                mask[first + i] = mask[first + int(torch.randint(0, i, (1,), generator=g))]
            if i < width:
                mask[first + i, i] = True
    return mask


def attend(batch, mask=None, scale=None, max_new=0, tile_rows=None, **more):
    """Runs the attention, compares every row with 64 bits, and requires that nothing else changed.  ``tile_rows`` None: every kernel."""
    import torch
    import frisk_b200 as F
    if tile_rows is None:
        return [attend(batch, mask, scale, max_new, n, **more) for n in (16, 128, 256, 0)][-1]
    out = torch.full((batch.rows,) + tuple(batch.q.shape[1:]), 77.0, dtype=batch.dtype, device="cuda")
    before = [bits(t) for t in batch.cache]
    got = F.cache_attention(batch.cache, batch.q, *batch.plan, mask=None if mask is None else mask.cuda(), scale=scale, max_new=max_new,
                            tile_rows=tile_rows, out=out, **more)
    F.cache_check()
    assert got is out
    assert all(torch.equal(a, bits(t)) for a, t in zip(before, batch.cache))
    ref, bound = co.attention(batch.cpu, batch.q.cpu(), *batch.host, mask=mask, scale=scale, terms=len(batch.cpu) == 4 and (tile_rows or batch.tile_rows(max_new)) > 16)
    got, inside = out.cpu().double(), batch.inside()
    assert bool((got[~inside] == 77.0).all())
    finite = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got) | ~inside[:, None, None], finite | ~inside[:, None, None])
    use = finite & inside[:, None, None]
    off = ((got - ref).abs() - bound)[use]
    assert off.numel() == 0 or float(off.max()) <= 0, (float(off.max()), float((got - ref)[use].abs().max()))
    return out


# ------------------------------------------------------------------------------------------------ write and read
SHAPES = [([1], [0], 1, 64, 16), ([1, 1, 1], [15, 16, 31], 2, 128, 16), ([5, 0, 70, 1], [0, 9, 60, 129], 3, 64, 32),
          ([200, 33], [1, 300], 8, 128, 128), ([0, 0], [4, 0], 1, 64, 64), ([17] * 40, list(range(40)), 5, 64, 16), ([3], [2000], 20, 128, 1024)]


@pytest.mark.parametrize("counts,lengths,hkv,d,page", SHAPES)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("gap", [0, 2])
def test_write_and_read(counts, lengths, hkv, d, page, dtype, e4m3, gap):
    import torch
    import frisk_b200 as F
    dtype = getattr(torch, dtype)
    b = Batch(counts, lengths, hkv, 1, d, page, dtype, torch.float8_e4m3fn if e4m3 else None, 1, gap, fill=False)
    k, v = b.k.cpu(), b.v.cpu()
    want = co.write(b.cpu, k, v, *b.host)
    assert F.cache_write(b.cache, b.k, b.v, *b.plan) is b.cache
    F.cache_check()
    assert same(b.cache, want)
    out = tuple(torch.full((b.rows, hkv, d + 8), 3.0, dtype=dtype, device="cuda")[..., :d] for _ in range(2))
    F.cache_read(b.cache, *b.plan, b.rows, out=out)
    F.cache_check()
    for i, o in enumerate(out):
        ref = torch.full((b.rows, hkv, d), 3.0, dtype=torch.float64)
        x = co.values(want, i)
        for r, _, p, at in co.slots(*b.host, page):
            ref[r] = x[p, :, at]
        assert torch.equal(o.cpu(), ref.to(dtype))  # four bits: no rounding
    if b.rows:
        fresh = F.cache_read(b.cache, *b.plan, b.rows, dtype=dtype)
        assert all(torch.equal(a[b.inside()], o[b.inside()]) for a, o in zip(fresh, out))


def test_special_rows_are_quantised():
    import torch
    import frisk_b200 as F
    rows = [torch.zeros(64), torch.full((64,), 448.0), torch.full((64,), 449.0), torch.full((64,), 2.0 ** -133), torch.full((64,), 3.38e38),
            torch.linspace(-1, 1, 64), torch.full((64,), -0.0), torch.logspace(-20, 3, 64), torch.ones(64), torch.ones(64), torch.full((64,), 1.75),
            torch.tensor([448.0] + [17.0, 19.0, 25.0, 2.0 ** -10, 3 * 2.0 ** -10, 1.5 * 2.0 ** -9] * 10 + [1.0] * 3)]
    x = torch.stack(rows).to(torch.bfloat16)
    x[8, 5], x[9, 63] = math.inf, math.nan
    x = x[:, None].repeat(1, 2, 1)
    n = len(rows)
    cache = F.paged_cache(2, 2, 16, 64, torch.float8_e4m3fn)
    plan = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([[1]], [0, n], [0])]
    F.cache_write(cache, x.cuda(), x.flip(0).cuda(), *plan)
    host = [t.cpu() for t in plan]
    want = co.write(tuple(t.cpu() * 0 if t.dtype == torch.uint8 else torch.zeros_like(t, device="cpu") for t in cache), x, x.flip(0), *host)
    assert same(cache, want)
    k, _ = F.cache_read(cache, *plan, n)
    k = k.cpu()
    assert k.dtype == torch.bfloat16 and bool(torch.isnan(k[8:10]).all()) and bool(torch.isfinite(k[:8]).all()) and bool(torch.isfinite(k[10:]).all())
    # half precision at its end: 65504 becomes 65536 in four bits, and is read as the largest finite value
    y = torch.full((1, 2, 64), 65504.0, dtype=torch.float16, device="cuda")
    plan[1][1] = 1
    F.cache_write(cache, y, -y, *plan)
    k, v = F.cache_read(cache, *plan, 1, dtype=torch.float16)
    assert bool((k == 65504).all()) and bool((v == -65504).all())


# ------------------------------------------------------------------------------------------------ attention
ATTEND = [  # counts, lengths, key heads, group, d, page
    ([1], [0], 1, 1, 64, 16), ([1], [200], 2, 4, 128, 16), ([1] * 5, [0, 1, 63, 64, 65], 1, 8, 64, 16), ([3, 1, 0, 7], [1000, 63, 5, 0], 2, 3, 128, 32),
    ([64, 60], [77, 500], 1, 2, 64, 64), ([5, 4], [64, 4000], 4, 5, 128, 128), ([17], [15], 1, 16, 64, 1024), ([33, 1, 2], [127, 300, 0], 2, 1, 128, 16),
    ([100], [250], 1, 8, 128, 64), ([1], [70000], 1, 1, 64, 256), ([2] * 70, [31 * i % 257 for i in range(70)], 1, 2, 64, 16), ([130], [0], 2, 4, 64, 32)]


@pytest.mark.parametrize("counts,lengths,hkv,group,d,page", ATTEND)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("scales", [None, (120, 134), (116, 122)])  # of an 8-bit cache: far apart, near each other
def test_attention(counts, lengths, hkv, group, d, page, dtype, scales):
    import torch
    held = torch.float8_e4m3fn if scales else None
    b = Batch(counts, lengths, hkv, group, d, page, getattr(torch, dtype), held, 3, gap=1, scales=scales or (0, 1))
    for n in (16, 128, 256):
        assert torch.equal(bits(attend(b, tile_rows=n)), bits(attend(b, tile_rows=n)))
    attend(b, mask=tree(b, 1))
    attend(b, mask=tree(b, 2, "random"), max_new=max(counts))
    attend(b, mask=tree(b, 4, width=max(1, max(counts) // 2)), max_new=1, scale=0.31)


@pytest.mark.parametrize("dtype,held", [("bfloat16", None), ("float16", "float8_e4m3fn")])
@pytest.mark.parametrize("count,group,d,length", [(1, 1, 64, 9001), (1, 3, 128, 5000), (5, 1, 128, 4999), (3, 3, 64, 300), (11, 1, 64, 7000), (29, 5, 128, 6007)])
def test_one_long_sequence(count, group, d, length, dtype, held):
    """One key head: the parts of many CTAs are joined, shared among the warps where rows are few."""
    import torch
    batch = Batch([count], [length], 1, group, d, 16, getattr(torch, dtype), held and getattr(torch, held), 9)
    attend(batch)
    attend(batch, mask=tree(batch, 13))


@pytest.mark.parametrize("e4m3", [False, True])
def test_rows_that_see_nothing_are_zero(e4m3):
    import torch
    for count in (6, 20, 40):
        b = Batch([count, 3], [0, 0], 2, 4, 64, 16, torch.float16, torch.float8_e4m3fn if e4m3 else None, 5)
        out = attend(b, mask=torch.zeros(b.rows, 4, dtype=torch.bool))
        assert not out.any()
        mask = torch.zeros(b.rows, count, dtype=torch.bool)
        mask[2, 1] = True
        out = attend(b, mask=mask)
        assert out[2].any() and not out[:2].any() and not out[3:].any()
        assert not attend(b, mask=torch.zeros(b.rows, 0, dtype=torch.bool)).any()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("count", [4, 20, 40])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, e4m3, count):
    """Keys and values of new tokens that are infinite, NaN or large: rows that see them get what the formula gives."""
    import torch
    b = Batch([count, 2], [70, 0], 1, 4, 128, 16, getattr(torch, dtype), torch.float8_e4m3fn if e4m3 else None, 6)
    table = b.table_cpu

    def at(i, ahead):
        pos = b.lengths[i] + ahead
        return int(table[i, pos // 16]), 0, pos % 16
    cpu = [t.clone() for t in b.cpu]
    if e4m3:
        cpu[2][at(0, 1)] = 255                                  # a key that was NaN
        cpu[3][at(0, 2)] = 255                                  # values that were
        cpu[3][at(0, 3)] = 250                                  # large values
        cpu[1].view(torch.uint8)[at(1, 1)][7] = 0x7f             # a code that is NaN
    else:
        cpu[0][at(0, 1)][3] = math.nan
        cpu[1][at(0, 2)][5] = math.inf
        cpu[1][at(0, 2)][6] = math.nan
        cpu[1][at(0, 3)][7] = -math.inf
        cpu[1][at(0, 3)][5] = -math.inf
        cpu[1][at(1, 1)][9] = math.nan
        cpu[0][at(1, 0)][9] = math.inf
    b.cpu = tuple(cpu)
    b.refresh()
    mask = torch.zeros(b.rows, count, dtype=torch.bool)
    mask[torch.arange(count), torch.arange(count)] = True
    mask[3, 2] = True
    mask[count, 0] = mask[count + 1, 1] = True
    mask[0, 0] = False
    out = attend(b, mask=mask)
    assert bool(torch.isfinite(out[0]).all())
    attend(b)


@pytest.mark.parametrize("e4m3", [False, True])
def test_wide_ranges_of_scores_and_values(e4m3):
    import torch
    for count in (1, 3, 12, 40, 130):
        b = Batch([count], [300], 1, 2, 64, 32, torch.bfloat16, torch.float8_e4m3fn if e4m3 else None, 7)
        cpu = [t.clone() for t in b.cpu]
        g = torch.Generator().manual_seed(1)
        if e4m3:  # scales from 2^-60 to 2^60, token by token
            cpu[3] = torch.where(cpu[3] == 255, cpu[3], torch.randint(67, 188, cpu[3].shape, generator=g).to(torch.uint8))
            cpu[2] = torch.where(cpu[2] == 255, cpu[2], torch.randint(110, 136, cpu[2].shape, generator=g).to(torch.uint8))
        else:
            cpu[1] = (cpu[1].double() * torch.exp2(torch.randint(-60, 61, cpu[1].shape[:3], generator=g).double())[..., None]).to(torch.bfloat16)
            cpu[0] = (cpu[0].double() * torch.exp2(torch.randint(-8, 5, cpu[0].shape[:3], generator=g).double())[..., None]).to(torch.bfloat16)
        b.cpu = tuple(cpu)
        b.refresh()
        attend(b)
        attend(b, scale=0.0)
        attend(b, scale=-0.2)
        b.q *= 1e-30
        attend(b)


def test_more_sequences_than_threads_and_strided_tables():
    import torch
    b = Batch([1] * 700, [7 * i % 50 for i in range(700)], 1, 1, 64, 16, torch.float16, None, 8)
    attend(b)
    wide = torch.full((700, 40), -9, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + b.plan[0].shape[1]] = b.plan[0]
    b.plan = (wide[:, 3:],) + b.plan[1:]
    attend(b)


def test_offsets_beyond_32_bits():
    """Pages more than 2^32 bytes into the cache."""
    import torch
    import frisk_b200 as F
    for dtype, e4m3 in ((torch.bfloat16, False), (torch.float16, True)):
        pages = 1 << 12 if not e4m3 else 1 << 13
        shape = (pages, 8, 1024, 128)  # 8 GiB each
        held = torch.float8_e4m3fn if e4m3 else dtype
        cache = tuple(torch.zeros(shape, dtype=torch.uint8 if e4m3 else dtype, device="cuda").view(held) for _ in range(2))
        if e4m3:
            cache += tuple(torch.zeros(shape[:3], dtype=torch.uint8, device="cuda") for _ in range(2))
        n = 1030
        g = torch.Generator().manual_seed(1)
        k, v, q = (torch.randn(n, 8, 128, generator=g).to(dtype).cuda() for _ in range(3))
        plan = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([[pages - 1, pages - 3]], [0, n], [0])]
        F.cache_write(cache, k, v, *plan)
        k2, v2 = F.cache_read(cache, *plan, n, dtype=dtype)
        small = tuple(t[pages - 3:].clone() for t in cache)
        back = F.cache_read(small, plan[0] - (pages - 3), *plan[1:], n, dtype=dtype)
        assert torch.equal(k2, back[0]) and torch.equal(v2, back[1]) and (e4m3 or torch.equal(k2, k))
        assert not any(bits(t[:4]).any() for t in cache)
        last = [torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([n - 3], dtype=torch.int32, device="cuda")]
        a = F.cache_attention(cache, q[-3:], plan[0], *last)
        c = F.cache_attention(small, q[-3:], plan[0] - (pages - 3), *last)
        F.cache_check()
        assert torch.equal(a, c) and bool(torch.isfinite(a).all()) and a.any()
        del cache


def test_tables_out_of_range_are_left_out_and_reported():
    import torch
    import frisk_b200 as F

    def run(table, starts, lengths, rows=8):
        cache = F.paged_cache(4, 1, 16, 64, torch.float16)
        x = torch.ones(rows, 1, 64, dtype=torch.float16, device="cuda")
        plan = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in (table, starts, lengths)]
        F.cache_write(cache, x, x, *plan)
        with pytest.raises(RuntimeError):
            F.cache_check()
        back = tuple(torch.full_like(x, 5.0) for _ in range(2))
        F.cache_read(cache, *plan, rows, out=back)
        with pytest.raises(RuntimeError):
            F.cache_check()
        out = torch.full_like(x, 5.0)
        F.cache_attention(cache, x, *plan, out=out)
        with pytest.raises(RuntimeError):
            F.cache_check()
        F.cache_check()  # (and clean again)
        return cache, back[0][:, 0, 0].tolist(), out[:, 0, 0].tolist()

    good = [1.0] * 4
    # a page that the cache does not have: only its rows are left out, the sequence's attention is undefined
    cache, back, out = run([[0], [4]], [0, 4, 8], [0, 0])
    assert back == good + [5.0] * 4 and out[:4] == good
    cache, back, out = run([[-1], [2]], [0, 4, 8], [0, 0])
    assert back == [5.0] * 4 + good and out[4:] == good
    assert int(cache[0][:2].ne(0).sum()) == 0
    # a negative length, more keys than the table holds
    assert run([[0], [1]], [0, 4, 8], [0, -1])[1:] == (good + [5.0] * 4,) * 2
    assert run([[0], [1]], [0, 4, 8], [13, 0])[1:] == ([5.0] * 4 + good,) * 2
    assert run([[0], [1]], [0, 4, 8], [2 ** 31 - 1, 0])[1:] == ([5.0] * 4 + good,) * 2
    # starts behind the rows
    assert run([[0], [1]], [0, 4, 9], [0, 0])[1:] == (good + [5.0] * 4,) * 2


def test_sequences_that_share_rows_do_not_overflow_the_plan():
    """Starts that descend again and again: twenty sequences of all rows, whose work counted in 32 bits would begin anew."""
    import torch
    import frisk_b200 as F
    rows, width, page = 65536, 4096, 1024
    cache = F.paged_cache(1, 1, page, 64, torch.float16)
    table = torch.zeros(40, width, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, rows] * 20 + [0], dtype=torch.int32, device="cuda")
    lengths = torch.full((40,), 4000000, dtype=torch.int32, device="cuda")
    q = torch.zeros(rows, 1, 64, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 5.0)
    F.cache_attention(cache, q, table, starts, lengths, tile_rows=16, out=out)
    with pytest.raises(RuntimeError):
        F.cache_check()
    assert bool((out == 5.0).all())


def test_a_mask_without_columns_takes_no_memory():
    """Tables and results in one buffer: the mask's rows have nothing that the results could overlap."""
    import torch
    import frisk_b200 as F
    rows, d = 600, 64
    buffer = torch.zeros(256 + rows * d * 2, dtype=torch.uint8, device="cuda")
    starts, lengths, table = (buffer[a:a + 4 * n].view(torch.int32) for a, n in ((0, 2), (8, 1), (16, 40)))
    starts[1], lengths[0] = rows, 7
    table.copy_(torch.arange(40))
    out = buffer[256:].view(torch.float16).view(rows, 1, d)
    cache = F.paged_cache(40, 1, 16, d, torch.float16)
    cache[1].fill_(2.0)
    q = torch.randn(rows, 1, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    F.cache_attention(cache, q, table.view(1, 40), starts, lengths, mask=torch.empty(rows, 0, dtype=torch.bool, device="cuda"), out=out)
    F.cache_check()
    assert bool((out == 2.0).all())


def test_captured_step_replayed_with_other_contents():
    """Rotate, write, attend: captured once, replayed as the sequences grow; two graphs at once; and step by step without a graph."""
    import torch
    import frisk_b200 as F
    hkv, group, d, page = 2, 4, 64, 16
    for held in (torch.bfloat16, torch.float8_e4m3fn):
        def new():
            cache = F.paged_cache(40, hkv, page, d, held)
            table = torch.randperm(40, generator=torch.Generator().manual_seed(2)).int().view(4, 10).cuda()
            return cache, table
        f, _ = F.rotary_frequencies(d)
        starts = torch.tensor([0, 3, 4, 6, 9], dtype=torch.int32, device="cuda")
        counts = starts[1:] - starts[:-1]

        def step(cache, table, lengths, positions, buf):
            q, k, v = buf[:, :8], buf[:, 8:10], buf[:, 10:]
            q, k = F.rotary(q, k, positions, f)
            F.cache_write(cache, k, v, table, starts, lengths)
            return F.cache_attention(cache, q, table, starts, lengths)

        inputs = [torch.randn(9, 12, d, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(12)]
        owner = torch.repeat_interleave(torch.arange(4, device="cuda"), counts.long())
        within = torch.arange(9, device="cuda") - starts[:-1].long()[owner]

        def all_steps(call, lengths, positions, buf):
            outs = []
            lengths.zero_()
            for x in inputs:
                positions.copy_(lengths.long()[owner] + within)
                buf.copy_(x)
                outs.append(call().clone())
                lengths += counts
            return torch.stack(outs)

        states = []
        for _ in range(3):
            cache, table = new()
            lengths = torch.zeros(4, dtype=torch.int32, device="cuda")
            positions, buf = torch.zeros(9, dtype=torch.int64, device="cuda"), inputs[0].clone()
            states.append((cache, table, lengths, positions, buf))
        plain = all_steps(lambda: step(*states[0]), *states[0][2:])
        F.cache_check()
        graphs, results = [], []
        for s in states[1:]:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                results.append(step(*s))
            graphs.append(graph)
            for t in s[0]:
                t.zero_()
        one = all_steps(lambda: (graphs[0].replay(), results[0])[1], *states[1][2:])
        assert torch.equal(plain, one)
        # both graphs, each on a stream of its own, at the same time
        for t in states[1][0]:
            t.zero_()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        got = [[], []]
        for s in states[1:]:
            s[2].zero_()
        torch.cuda.synchronize()
        for x in inputs:
            for n, s in enumerate(states[1:]):
                with torch.cuda.stream(streams[n]):
                    s[3].copy_(s[2].long()[owner] + within)
                    s[4].copy_(x)
                    graphs[n].replay()
                    got[n].append(results[n].clone())
                    s[2].add_(counts)
        torch.cuda.synchronize()
        assert torch.equal(plain, torch.stack(got[0])) and torch.equal(plain, torch.stack(got[1]))
        F.cache_check()
        # the last step's result against 64 bits
        cache, table, lengths, positions, buf = states[0]
        q, _ = F.rotary(buf[:, :8], buf[:, 8:10], positions, f)
        ref, bound = co.attention(tuple(t.cpu() for t in cache), q.cpu(), table.cpu(), starts.tolist(), (lengths - counts).tolist())
        assert bool(((plain[-1].cpu().double() - ref).abs() <= bound).all())


def test_calls_on_two_streams_at_once():
    import torch
    import frisk_b200 as F
    a = Batch([3, 5], [3000, 100], 4, 4, 128, 64, torch.bfloat16, None, 11)
    b = Batch([20, 1], [900, 5000], 4, 4, 128, 64, torch.bfloat16, torch.float8_e4m3fn, 12)
    want = [F.cache_attention(x.cache, x.q, *x.plan) for x in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s, x in zip(streams, (a, b)):
            got.append(F.cache_attention(x.cache, x.q, *x.plan, stream=s))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))
    F.cache_check(stream=streams[0])


def test_refusals():
    import torch
    import frisk_b200 as F
    b = Batch([3], [20], 2, 2, 64, 16, torch.float16, None, 1)
    e = Batch([3], [20], 2, 2, 64, 16, torch.float16, torch.float8_e4m3fn, 1)
    t, s, n = b.plan
    odd = torch.zeros(3 * 2 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(3, 2, 64)
    for bad in (
            lambda: F.cache_write(b.cache, b.k.bfloat16(), b.v.bfloat16(), *b.plan), lambda: F.cache_write(b.cache, b.k, b.v[:2], *b.plan),
            lambda: F.cache_write(b.cache, odd, b.v, *b.plan), lambda: F.cache_write(e.cache, b.k.float(), b.v.float(), *b.plan),
            lambda: F.cache_write(e.cache[:2], b.k, b.v, *b.plan), lambda: F.cache_write((b.cache[0], b.cache[1][:, :1]), b.k, b.v, *b.plan),
            lambda: F.cache_write((b.cache[0], b.cache[0]), b.k, b.v, *b.plan), lambda: F.cache_write(b.cache, b.k, b.v, t.long(), s, n),
            lambda: F.cache_write(b.cache, b.k, b.v, t, s[:1], n), lambda: F.cache_write(b.cache, b.k, b.v, t, s.cpu(), n),
            lambda: F.cache_write(b.cache, b.cache[0].view(-1, 2, 64)[:3], b.v, *b.plan), lambda: F.cache_read(b.cache, *b.plan, 3, dtype=torch.bfloat16),
            lambda: F.cache_read(b.cache, *b.plan, 3, out=(b.k, b.k)), lambda: F.cache_read(b.cache, *b.plan, 4, out=(b.k, b.v)),
            lambda: F.cache_read(e.cache, *b.plan, 3, dtype=torch.float32), lambda: F.cache_attention(b.cache, b.q.bfloat16(), *b.plan),
            lambda: F.cache_attention(b.cache, b.q[:, :3], *b.plan), lambda: F.cache_attention(b.cache, b.q, *b.plan, out=b.q),
            lambda: F.cache_attention(b.cache, b.q, *b.plan, scale=math.nan), lambda: F.cache_attention(b.cache, b.q, *b.plan, mask=torch.ones(3, 3, device="cuda")),
            lambda: F.cache_attention(b.cache, b.q, *b.plan, mask=torch.ones(2, 3, device="cuda").bool()),
            lambda: F.cache_attention(b.cache, b.q, *b.plan, out=torch.empty(3, 4, 128, device="cuda").half()[..., ::2])):
        with pytest.raises(ValueError):
            bad()
    F.cache_check()


def test_the_current_device_and_an_empty_batch():
    import torch
    import frisk_b200 as F
    b = Batch([2], [5], 1, 1, 64, 16, torch.float16, None, 1)
    empty = [torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")]
    out = torch.full_like(b.q, 4.0)
    F.cache_attention(b.cache, b.q, *empty, out=out)
    F.cache_write(b.cache, b.k, b.v, *empty)
    assert bool((out == 4).all())
    none = F.cache_attention(b.cache, b.q[:0], b.plan[0], torch.zeros_like(b.plan[1]), b.plan[2])
    assert none.shape[0] == 0
    assert torch.cuda.current_device() == 0
    F.cache_check()
