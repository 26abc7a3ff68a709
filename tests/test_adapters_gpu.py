"""Low-rank adapters of many requests against oracle/serving_oracle.py, which derives the bounds."""
import math

import pytest

from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu


class Requests:
    def __init__(self, counts, k, n, rank, count, dtype="bfloat16", wide=False, seed=0, gap=0, pitch=0, odd=0, size=1.0):
        """``pitch``: more elements between rows; ``odd``: columns in front of c in its buffer."""
        import torch
        g = torch.Generator().manual_seed(seed)
        self.dtype = dt = getattr(torch, dtype)
        self.starts = [gap]
        for m in counts:
            self.starts.append(self.starts[-1] + m)
        self.rows = rows = self.starts[-1] + gap

        def held(shape, scale, front=0, more=0, to=dt):
            cols = -(-(shape[-1] + front + more) // 8) * 8 if not front else shape[-1] + front + more
            whole = torch.full(shape[:-1] + (cols,), math.nan, dtype=to)
            whole[..., front:front + shape[-1]] = (torch.randn(shape, generator=g) * scale).to(to)
            return whole

        self.whole = [held((rows, k), size, more=pitch), held((count, rank, k), k ** -0.5, more=pitch), held((count, n, rank), 0.7, more=pitch),
                      held((rows, n), 1.0, front=odd, more=pitch, to=torch.float32 if wide else dt)]
        self.cut = [slice(0, k), slice(0, k), slice(0, rank), slice(odd, odd + n)]
        self.which = [int(torch.randint(-1, count, (1,), generator=g)) if count else -1 for _ in counts]
        self.scales = torch.rand(count, generator=g) * 2 - 1
        self.cpu = [t[..., s] for t, s in zip(self.whole, self.cut)]

    def run(self, scales=True, in_place=False, out=None, stream=None):
        import torch
        import frisk_b200 as F
        wholes = [t.cuda() for t in self.whole]
        x, a, b, c = (t[..., s] for t, s in zip(wholes, self.cut))
        starts, which = torch.tensor(self.starts, dtype=torch.int32).cuda(), torch.tensor(self.which, dtype=torch.int32).cuda()
        scales = self.scales.cuda() if scales else None
        if in_place:
            out = c
        elif out is None:
            out = torch.full(c.shape, 55.0, dtype=c.dtype, device="cuda")
        got = F.adapter_gemm(x, a, b, c, starts, which, scales=scales, out=out, stream=stream)
        if stream is not None:
            stream.synchronize()
        F.cache_check()
        assert got is out
        if in_place:  # what is beside c stays as it was
            left = [torch.equal(wholes[3][:, s].cpu().view(torch.uint8), self.whole[3][:, s].view(torch.uint8)) for s in (slice(0, self.cut[3].start), slice(self.cut[3].stop, None))]
            assert all(left)
        return got

    def check(self, scales=True, in_place=False, **more):
        import torch
        got = self.run(scales, in_place, **more).cpu().double()  # (``out`` of another's holds 55 where nothing is written)
        want, bound = so.adapters(*self.cpu, self.starts, self.which, self.scales if scales else None)
        inside = torch.zeros(self.rows, dtype=torch.bool)
        inside[self.starts[0]:self.starts[-1]] = True
        outside = self.cpu[3].double()[~inside] if in_place else torch.full(want[~inside].shape, 55.0, dtype=torch.float64)
        assert torch.equal(got[~inside], outside)
        finite = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got)[inside], finite[inside])
        off = ((got - want).abs() - bound)[inside[:, None] & finite]
        assert off.numel() == 0 or float(off.max()) <= 0, (float(off.max()), float((got - want)[inside].abs().max()))


@pytest.mark.parametrize("counts", [[1], [1] * 9, [0, 3, 16, 0, 17, 1], [40, 5, 33], [64], [128, 1], [129, 300], [3] * 300, [200, 0, 1, 130, 77, 128], [300, 129, 200], [640]])
@pytest.mark.parametrize("k,n,rank", [(64, 32, 8), (72, 100, 16), (8, 8, 24), (1, 1, 8), (250, 333, 32), (1000, 96, 40), (513, 520, 64), (300, 70, 128), (33, 31, 72)])
@pytest.mark.parametrize("dtype,wide", [("bfloat16", False), ("bfloat16", True), ("float16", False), ("float16", True)])
def test_adapters(counts, k, n, rank, dtype, wide):
    r = Requests(counts, k, n, rank, 5, dtype, wide, seed=k + len(counts), gap=len(counts) % 3, pitch=8 * (n % 2), odd=n % 4)
    r.check()
    r.check(scales=False, in_place=True)


SHARED = [[1] * 256, [1] * 257, [2, 0, 1] * 400, [1] * 2049, [0, 1, 3, 2] * 50, [5] * 90 + [40], [47] * 50, [0] * 255 + [17], [1, 70, 30] * 30]


@pytest.mark.parametrize("counts", SHARED, ids=range(len(SHARED)))
@pytest.mark.parametrize("k,n,rank,count", [(250, 333, 8, 3), (64, 40, 16, 1), (520, 96, 64, 2), (72, 130, 104, 40)])
@pytest.mark.parametrize("dtype,wide", [("bfloat16", False), ("float16", True)])
def test_sequences_that_share_adapters(counts, k, n, rank, count, dtype, wide):
    """Many sequences of few adapters, which come together by adapter, in every mixture."""
    import torch
    r = Requests(counts, k, n, rank, count, dtype, wide, seed=rank, gap=2, pitch=8, odd=n % 4)
    r.check()
    r.check(in_place=True)
    r.which = [0] * len(counts)
    r.check(scales=False)
    r.which = [(7 * i) % (count + 1) - 1 for i in range(len(counts))]
    plain = r.run().cpu()
    # what is not finite stays in its row
    last = r.starts[-1] - 1
    r.whole[0][last, :k] = math.nan
    got = r.run().cpu()
    assert torch.equal(got[:last], plain[:last]) and torch.equal(got[last + 1:], plain[last + 1:])


def test_many_requests_replayed():
    """A captured call with other adapters and other numbers of rows, and tables out of range."""
    import torch
    import frisk_b200 as F
    r = Requests([1] * 200, 200, 96, 16, 3, seed=2)
    x, a, b, c = (t.cuda()[..., s] for t, s in zip(r.whole, r.cut))
    starts, which, scales = torch.tensor(r.starts, dtype=torch.int32).cuda(), torch.tensor(r.which, dtype=torch.int32).cuda(), r.scales.cuda()
    out = torch.full_like(c, 55.0)
    graph = torch.cuda.CUDAGraph()
    F.adapter_gemm(x, a, b, c, starts, which, scales=scales, out=out)
    with torch.cuda.graph(graph):
        F.adapter_gemm(x, a, b, c, starts, which, scales=scales, out=out)
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        cut = [0] + sorted(torch.randint(0, 201, (199,), generator=g).tolist()) + [200]
        now = torch.randint(-1, 3, (200,), generator=g).tolist()
        which.copy_(torch.tensor(now, dtype=torch.int32))
        starts.copy_(torch.tensor(cut, dtype=torch.int32))
        out.fill_(55.0)
        graph.replay()
        F.cache_check()
        want, bound = so.adapters(*r.cpu, cut, now, r.scales)
        assert float(((out.cpu().double() - want).abs() - bound).max()) <= 0
    good = out.clone()
    bad = list(cut)
    bad[100] = -5  # sequences 99 and 100 have no rows
    bad_which = list(now)
    bad_which[0:3] = [3, 1 << 30, -9]
    which.copy_(torch.tensor(bad_which, dtype=torch.int32))
    starts.copy_(torch.tensor(bad, dtype=torch.int32))
    out.fill_(55.0)
    graph.replay()
    with pytest.raises(RuntimeError, match="table"):
        F.cache_check()
    assert torch.equal(out[:cut[3]], c[:cut[3]]) and torch.equal(out[cut[3]:cut[99]], good[cut[3]:cut[99]]) and torch.equal(out[cut[101]:], good[cut[101]:])
    assert bool((out[cut[99]:cut[101]] == 55.0).all())
    # all rows again and again: more than there are tiles for
    starts.copy_(torch.tensor([0, 200] * 100 + [0], dtype=torch.int32))
    which.fill_(1)
    graph.replay()
    with pytest.raises(RuntimeError, match="table"):
        F.cache_check()
    want, bound = so.adapters(*r.cpu, [0, 200], [1], r.scales)
    assert float(((out.cpu().double() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("counts", [[3, 0, 17], [300, 129, 200]])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("c_at,out_at,n", [(0, 1, 64), (1, 0, 64), (0, 8, 136), (3, 5, 37), (8, 0, 130), (0, 2, 2), (1, 1, 1)])
def test_results_elsewhere(counts, wide, c_at, out_at, n):
    """c and the result begin at other places of 16 bytes; what is beside the result, and behind the last row, stays."""
    import torch
    r = Requests(counts, 72, n, 16, 3, "bfloat16", wide, seed=n, gap=1, odd=c_at)
    buf = torch.full((r.rows, n + out_at + 7), 55.0, dtype=r.whole[3].dtype, device="cuda")
    r.check(out=buf[:, out_at:out_at + n])
    buf[:, out_at:out_at + n] = 55.0
    assert bool((buf == 55.0).all())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_longer_sums(dtype):
    for wide in (False, True):
        Requests([2, 1, 30, 200], 5000, 2500, 16, 3, dtype, wide, seed=1).check()
        Requests([70, 90], 4096, 1024, 64, 2, dtype, wide, seed=2).check()


def test_sums_beyond_fp16():
    """x A^T of 10^6 and B of 10^-5: terms stand at a power of two of their row; and the other way round."""
    for size, weight in ((3.0e4, 1e-4), (8.0e3, 1e-4), (1e-4, 300.0)):  # (the first has infinities in most rows of x)
        r = Requests([5, 40], 512, 64, 16, 2, "float16", True, seed=3, size=size)
        r.whole[2] *= weight
        r.whole[1][:, 0] *= 2.0 ** 6   # rows hold large and small sums side by side
        r.cpu = [t[..., s] for t, s in zip(r.whole, r.cut)]
        r.check()
        assert size > 1e4 or float(r.run().abs().max()) < math.inf


def test_what_is_not_finite_stays_in_its_row():
    import torch
    for dtype in ("bfloat16", "float16"):
        r = Requests([4, 3, 20], 200, 96, 16, 3, dtype, seed=6)
        r.which = [0, 1, 2]
        plain = r.run().cpu()
        for value in (math.nan, math.inf, -math.inf):
            r.whole[0][1, 7] = value
            r.whole[0][10, 199] = value
            got = r.run().cpu()
            hit = torch.zeros(27, dtype=torch.bool)
            hit[[1, 10]] = True
            assert not torch.isfinite(got[hit]).any()
            assert torch.equal(got[~hit], plain[~hit])
        # and a weight of another adapter than the row's
        r = Requests([4, 3, 20], 200, 96, 16, 3, dtype, seed=6)
        r.which = [0, 0, 2]
        plain = r.run().cpu()
        r.whole[1][1], r.whole[2][1] = math.nan, math.inf
        assert torch.equal(r.run().cpu(), plain)


@pytest.mark.parametrize("batch,new", [(80, 128), (2, 300), (64, 1), (130, 20)])
@pytest.mark.parametrize("rank", [16, 128])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_long_sums(dtype, rank, batch, new):
    """32-bit results of an inner index of 8192.  Tensor cores cut what an addition leaves below 24 bits: less than 2 u of the accumulator, u = 2^-24.  In the norm
    over all results, where a sum's beginning is no larger than the sum, chains of 8 additions are off by at most 16 u, in two products 32 u; the terms that a
    sum becomes leave 4 u, and adding up 64 parts, each time rounded by u, in random directions, 8 u.  (One chain over half of the index would be off by 256 u and more.)"""
    import torch
    import frisk_b200 as F
    k, n, t = 8192, 256, getattr(torch, dtype)
    torch.manual_seed(rank + batch)
    x, a, b = torch.randn(batch * new, k, device="cuda").to(t), torch.randn(2, rank, k, device="cuda").to(t), torch.randn(2, n, rank, device="cuda").to(t)
    starts, which = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * new, torch.arange(batch, dtype=torch.int32, device="cuda") % 2
    got = F.adapter_gemm(x, a, b, torch.zeros(batch * new, n, device="cuda"), starts, which).double()
    F.cache_check()
    for w in range(2):
        rows = (which == w).repeat_interleave(new)
        want = x[rows].double() @ a[w].double().t() @ b[w].double().t()
        assert float((got[rows] - want).norm() / want.norm()) <= 44 * 2.0 ** -24


def test_the_same_result_every_time():
    import torch
    r = Requests([1, 5, 70, 200, 0, 3], 1500, 700, 32, 4, seed=8)
    first = r.run()
    for _ in range(3):
        assert torch.equal(r.run(), first)


@pytest.mark.parametrize("new", [35, 7000])
def test_offsets_beyond_32_bits(new):
    """Rows of c and the result behind the first 2^31 elements, and adapters behind them: as those by themselves."""
    import torch
    import frisk_b200 as F
    rows, k, n, t = 70000, 64, 32768, torch.bfloat16
    torch.manual_seed(new)
    x, a, b = torch.randn(rows, k, device="cuda").to(t), torch.randn(2, 16, k, device="cuda").to(t), torch.randn(2, n, 16, device="cuda").to(t)
    c = torch.zeros(rows, n, dtype=t, device="cuda")
    c[-new:] = torch.randn(new, n, device="cuda").to(t)
    starts = torch.arange(rows // new + 1, dtype=torch.int32, device="cuda") * new
    which = torch.arange(rows // new, dtype=torch.int32, device="cuda") % 2
    got = F.adapter_gemm(x, a, b, c, starts, which)
    few = F.adapter_gemm(x[-new:].clone(), a, b, c[-new:].clone(), starts[:2], which[-1:])
    assert torch.equal(got[-new:], few)
    del c, got
    a = torch.zeros(20000, 16, 8192, dtype=t, device="cuda")
    a[-1] = torch.randn(16, 8192, device="cuda").to(t)
    x = torch.randn(new, 8192, device="cuda").to(t)
    b = torch.randn(20000, 8, 16, device="cuda").to(t)
    c = torch.zeros(new, 8, device="cuda")
    got = F.adapter_gemm(x, a, b, c, starts[:2], which[:1] * 0 + 19999)
    few = F.adapter_gemm(x, a[-1:].clone(), b[-1:].clone(), c, starts[:2], which[:1] * 0)
    F.cache_check()
    assert torch.equal(got, few) and bool(got.any())


def test_tables_out_of_range():
    import torch
    import frisk_b200 as F
    r = Requests([3, 4, 2], 64, 40, 8, 2, seed=4)
    x, a, b, c = (t.cuda()[..., s] for t, s in zip(r.whole, r.cut))

    def says(starts, which, *weights):
        out = torch.full_like(c, 55.0)
        F.adapter_gemm(x, *(weights or (a, b)), c, torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(which, dtype=torch.int32).cuda(), out=out)
        with pytest.raises(RuntimeError, match="table"):
            F.cache_check()
        F.cache_check()
        return out

    out = says(r.starts, [0, 2, 1])
    assert torch.equal(out[3:7], c[3:7]) and not torch.equal(out[:3], c[:3])
    assert torch.equal(says(r.starts, [1 << 30, 0, -5])[:3], c[:3])
    assert torch.equal(says(r.starts, [0, -1, 0], a[:0], b[:0]), c)
    for starts in ([-1, 3, 7, 9], [0, 3, 2, 9], [0, 3, 7, 10], [0, 3, 1 << 30, 9], [0, 3, -(1 << 31), 9]):
        out = says(starts, [0, 1, 0])
        for s in range(3):
            lo, hi = starts[s], starts[s + 1]
            if 0 <= lo <= hi <= 9 and starts[s:s + 2] == [0, 3, 7, 9][s:s + 2]:
                assert not torch.equal(out[lo:hi], c[lo:hi])
    # long sequences: behind one out of range all rows come again, more tiles than there are places for
    r = Requests([1024, 0, 0], 64, 40, 8, 2, seed=5)
    x, a, b, c = (t.cuda()[..., s] for t, s in zip(r.whole, r.cut))
    starts, which = torch.tensor([0, 1024, 1024, 1024], dtype=torch.int32).cuda(), torch.tensor([1, 1, 1], dtype=torch.int32).cuda()
    want = F.adapter_gemm(x, a, b, c, starts, which)
    F.cache_check()
    assert torch.equal(says([0, 1024, 0, 1024], [1, 1, 1]), want)


def test_refusals():
    import torch
    import frisk_b200 as F
    x, a, b, c = torch.zeros(6, 64), torch.zeros(2, 16, 64), torch.zeros(2, 40, 16), torch.zeros(6, 40)
    x, a, b, c = (t.bfloat16().cuda() for t in (x, a, b, c))
    starts, which, scales = torch.tensor([0, 2, 6], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.ones(2).cuda()
    good = dict(x=x, a=a, b=b, c=c, starts=starts, adapters=which, scales=scales, out=None)
    F.adapter_gemm(**good)
    both = torch.zeros(6, 104, dtype=torch.bfloat16, device="cuda")
    F.adapter_gemm(**dict(good, x=both[:, :64], c=both[:, 64:], out=both[:, 64:]))  # columns of one buffer
    for change in (dict(x=x.half()), dict(x=x.float(), a=a.float(), b=b.float(), c=c.float()), dict(c=c.half()), dict(a=a[:1]), dict(a=a[:, :8]), dict(b=b[..., :8]), dict(x=x[:, :56]),
                   dict(c=c[:, :32]), dict(c=c[:5]), dict(starts=starts[:2]), dict(starts=starts.long()), dict(adapters=which.long()), dict(scales=scales[:1]),
                   dict(scales=scales.double()), dict(x=x.cpu()), dict(scales=scales.cpu()), dict(out=c.float()), dict(out=c[:, :32]),
                   dict(a=torch.zeros(2, 12, 64, device="cuda").bfloat16(), b=torch.zeros(2, 40, 12, device="cuda").bfloat16()),     # ranks
                   dict(a=torch.zeros(2, 136, 64, device="cuda").bfloat16(), b=torch.zeros(2, 40, 136, device="cuda").bfloat16()),
                   dict(x=torch.zeros(6, 65, device="cuda").bfloat16()[:, 1:]),                                                        # rows on 16 bytes
                   dict(a=torch.zeros(2, 16, 68, device="cuda").bfloat16()[..., :64]),
                   dict(x=both[:, :64], out=both[:, 40:80]), dict(out=both.view(-1)[:240].view(6, 40), x=both[:, :64]),               # overlaps
                   dict(c=both[:, :40], out=both[:, 8:48]), dict(out=torch.zeros(40, device="cuda").bfloat16().expand(6, 40))):
        with pytest.raises(ValueError):
            F.adapter_gemm(**dict(good, **change))
    empty = F.adapter_gemm(x[:0], a, b, c[:0], starts * 0, which)
    assert empty.shape == (0, 40)
    out = torch.full_like(c, 3.0)
    F.adapter_gemm(x, a, b, c, starts[:1], which[:0], out=out)  # no sequences: no row is anyone's
    assert bool((out == 3.0).all())
    F.cache_check()


def test_streams_and_graphs():
    import torch
    import frisk_b200 as F
    r = Requests([1, 5, 2], 256, 96, 16, 4, seed=12)
    r.check(stream=torch.cuda.Stream())
    x, a, b, c = (t.cuda()[..., s] for t, s in zip(r.whole, r.cut))
    starts, which, scales = torch.tensor(r.starts, dtype=torch.int32).cuda(), torch.tensor(r.which, dtype=torch.int32).cuda(), r.scales.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.adapter_gemm(x, a, b, c, starts, which, scales=scales)
    for now, cut in (([0, 1, 2], [0, 1, 6, 8]), ([3, -1, 3], [0, 4, 4, 8]), ([1, 2, 0], [0, 0, 8, 8])):
        which.copy_(torch.tensor(now, dtype=torch.int32))
        starts.copy_(torch.tensor(cut, dtype=torch.int32))
        graph.replay()
        F.cache_check()
        want, bound = so.adapters(*r.cpu, cut, now, r.scales)
        assert float(((out.cpu().double() - want).abs() - bound).max()) <= 0
