"""Low-rank adapters where the product cancels: the sums between the two products have to keep 32 bits, whatever the result's type."""
import pytest

pytestmark = pytest.mark.gpu


def lists(counts, which):
    import torch
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return torch.tensor(starts, dtype=torch.int32, device="cuda"), torch.tensor(which, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("counts", [[1], [3, 0, 17, 40], [1] * 300, [5] * 90, [128, 1, 130, 300], [700]])
@pytest.mark.parametrize("k,n,rank", [(64, 32, 8), (200, 100, 16), (72, 65, 40), (520, 130, 64), (1000, 200, 128)])
@pytest.mark.parametrize("dtype,wide", [("bfloat16", False), ("bfloat16", True), ("float16", False), ("float16", True)])
def test_sums_that_cancel(counts, k, n, rank, dtype, wide):
    cancelling(counts, k, n, rank, dtype, wide)


@pytest.mark.parametrize("counts", [[1], [3, 0, 17, 40], [700]])
@pytest.mark.parametrize("wide", [False, True])
def test_small_sums_that_cancel(counts, wide):
    """The same near the lower end of the range: sums of 2^-101, and weights that bring them back."""
    cancelling(counts, 200, 100, 16, "bfloat16", wide, 2.0 ** -116)


def cancelling(counts, k, n, rank, dtype, wide, size=1.0):
    """Sums of 24 bits, p 2^8 + q + u 2^-8 with p, q, u of 8 bits, of which a column takes the difference of two that are less than 2^-1 apart: exact in sums of 32 bits,
    in whatever order (every partial sum is a multiple of 2^-8 below 2^16), and so is the result in any type."""
    import torch
    import frisk_b200 as F
    dt, rows = getattr(torch, dtype), sum(counts)
    g = torch.Generator().manual_seed(rows + k)
    a, x = torch.zeros(3, rank, k), torch.zeros(rows, k)
    at = torch.randperm(k, generator=g)[:3]
    x[:, at] = torch.tensor([256.0, 1.0, 2.0 ** -8]) * size
    a[:, ::2, at] = torch.randint(0, 256, (3, rank // 2, 3), generator=g).float()
    a[:, ::2, at[0]] = torch.randint(128, 256, (3, rank // 2), generator=g).float()
    a[:, ::2, at[2]] = torch.randint(64, 128, (3, rank // 2), generator=g).float()
    a[:, 1::2] = a[:, ::2]
    a[:, 1::2, at[2]] += torch.randint(-64, 64, (3, rank // 2), generator=g).float()
    pair, sign = torch.randint(0, rank // 2, (3, n), generator=g), torch.randint(0, 2, (3, n), generator=g) * 2.0 - 1
    b = torch.zeros(3, n, rank)
    b.scatter_(2, (2 * pair)[..., None], sign[..., None]).scatter_(2, (2 * pair + 1)[..., None], -sign[..., None])
    x[::2] = -x[::2]
    b /= size
    c = torch.randint(-1, 2, (rows, n), generator=g).float() / 256
    which = [i % 3 for i in range(len(counts))]
    starts, adapters = lists(counts, which)
    got = F.adapter_gemm(x.to(dt).cuda(), a.to(dt).cuda(), b.to(dt).cuda(), c.to(torch.float32 if wide else dt).cuda(), starts, adapters)
    F.cache_check()
    of_row = torch.tensor(which).repeat_interleave(torch.tensor(counts))
    want = c.double()
    for w in range(3):
        mine = of_row == w
        want[mine] += x[mine].double() @ a[w].double().t() @ b[w].double().t()
    assert torch.equal(got.double().cpu(), want)


@pytest.mark.parametrize("rows,rank", [(1, 8), (20, 16), (520, 16), (520, 128)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_long_sums_that_cancel(dtype, rows, rank):
    """16-bit results of an inner index of 2^21 (2^17 where there are more rows), c being the rounded product.  Tensor cores cut what an addition leaves below 24 bits, less than 2 u of the
    accumulator, u = 2^-24, always towards zero.  A chain of 8 additions, and the 8 of the columns, are off by at most 16 u each; up to 256 parts of a warp, of positive values, are added up rounding to nearest in
    random directions, 256^1/2 u / 3^1/2 and six deviations of that 56 u; 64 parts of warps and CTAs in a tree of two sums of 8, 16 u at most.  In all 104 u of the product, and half a step of the
    result.  (Chains that are not cut short are off by some u / 3 each addition: at 2^21 in 64 warps by 700 u.)"""
    import torch
    import frisk_b200 as F
    dt, u, half = getattr(torch, dtype), 2.0 ** -24, 2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -11
    k, n = (1 << 21) if rows == 1 else (1 << 17), 40
    torch.manual_seed(rows)
    x = (torch.rand(rows, k, device="cuda") * 2.0 ** -9 + 2.0 ** -10).to(dt)
    a = (torch.rand(1, rank, k, device="cuda") + 0.5).to(dt)
    b = (torch.rand(1, n, rank, device="cuda") * 0.1 + 0.1).to(dt)
    product = sum(x[:, i:i + 65536].double() @ a[0, :, i:i + 65536].double().t() for i in range(0, k, 65536)) @ b[0].double().t()
    c = -product.to(dt)
    starts, adapters = lists([rows], [0])
    got = F.adapter_gemm(x, a, b, c, starts, adapters)
    F.cache_check()
    want = c.double() + product
    off = (got.double() - want).norm()
    assert float(off) <= half * float(want.norm()) + 104 * u * float(product.norm())


def by_definition(x, a, b, c, counts, which):
    """Element by element in 64 bits, so that infinities and NaN go the way of the formula."""
    import torch
    of_row = torch.tensor(which).repeat_interleave(torch.tensor(counts))
    out = c.double().clone()
    for w in range(len(a)):
        mine = of_row == w
        t = torch.stack([(x[mine].double() * row.double()).sum(-1) for row in a[w]], -1)
        out[mine] += torch.stack([(t * row.double()).sum(-1) for row in b[w]], -1)
    return out


@pytest.mark.parametrize("counts", [[6], [3, 0, 17, 40], [1] * 300, [128, 1, 130, 300]])
@pytest.mark.parametrize("k,n,rank", [(64, 37, 8), (72, 65, 40), (200, 130, 128)])
@pytest.mark.parametrize("dtype,wide", [("bfloat16", False), ("bfloat16", True), ("float16", False), ("float16", True)])
def test_infinite_weights(counts, k, n, rank, dtype, wide):
    """An infinite element of B makes its column infinite, by the sign of the sum that it weighs, and nothing else; one of A all that its sum reaches; 0 times it, and two of other signs, are NaN."""
    import torch
    import frisk_b200 as F
    from oracle import serving_oracle as so
    dt, rows, inf = getattr(torch, dtype), sum(counts), float("inf")
    g = torch.Generator().manual_seed(rows + n)
    # (sums beyond fp16's range, and what they weigh)
    x, a, b = torch.randn(rows, k, generator=g) * 100, torch.randn(3, rank, k, generator=g) * 100, torch.randn(3, n, rank, generator=g) * 0.01
    b[0, 3, 2], b[0, 5, 1], b[0, 5, 6], b[0, n - 1, rank - 1], b[1, 0, 0] = inf, inf, -inf, -inf, inf
    a[1, 3, 7], a[2, 4, k - 1], a[2, 5, 0] = inf, -inf, inf
    x[4::5] = 0
    x, a, b = x.to(dt), a.to(dt), b.to(dt)
    c = torch.randn(rows, n, generator=g).to(torch.float32 if wide else dt)
    which = [(i + 1) % 3 if len(counts) > 1 else 0 for i in range(len(counts))]
    starts, adapters = lists(counts, which)
    got = F.adapter_gemm(x.cuda(), a.cuda(), b.cuda(), c.cuda(), starts, adapters).double().cpu()
    F.cache_check()
    want = by_definition(x, a, b, c, counts, which)
    assert bool(want.isinf().any()) and bool(want.isnan().any()) and bool(want.isfinite().any())
    _, bound = so.adapters(x, a, b, c, starts.tolist(), which)
    most = torch.finfo(c.dtype).max
    finite = want.isfinite() & (want.abs() < most)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    assert float(((got - want).abs() - bound)[finite].max()) <= 0


@pytest.mark.parametrize("counts", [[2], [30, 3], [600]])
@pytest.mark.parametrize("wide", [False, True])
def test_sums_at_the_end_of_the_range(counts, wide):
    """Sums between bf16's largest value, 1.9921875 2^127, and that of 32 bits keep their value."""
    import torch
    import frisk_b200 as F
    rows = sum(counts)
    x, a, b = torch.zeros(rows, 64), torch.zeros(1, 8, 64), torch.zeros(1, 24, 8)
    x[:, :2] = torch.tensor([2.0 ** 63, 2.0 ** 60])
    a[:, :, :2] = torch.tensor([1.9921875 * 2.0 ** 64, 3 * 2.0 ** 58])  # the largest value, and 3 2^-9 of the power: 1.998046875 2^127
    a[:, 1::2] = -a[:, 1::2]
    b[:] = torch.arange(1, 9) * 2.0 ** -120
    x, a, b = (t.bfloat16().cuda() for t in (x, a, b))
    starts, adapters = lists(counts, [0] * len(counts))
    got = F.adapter_gemm(x, a, b, torch.zeros(rows, 24, dtype=torch.float32 if wide else torch.bfloat16, device="cuda"), starts, adapters)
    F.cache_check()
    want = 1.998046875 * -4 * 2.0 ** 7  # (the sum of 1 - 2 + 3 .. - 8 is -4)
    assert torch.equal(got.cpu(), torch.full((rows, 24), want, dtype=got.dtype))
