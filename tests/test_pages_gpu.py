"""Pages that sequences share against oracle/serving_oracle.py: tables to the last entry, caches to the last bit."""
import math
import random

import pytest

from oracle import cache_oracle as co
from oracle import serving_oracle as so
from tests.test_cache_gpu import Batch, bits, same

pytestmark = pytest.mark.gpu


def new_cache(pages, heads, page, d, held, seed=0):
    """Every byte of it another (codes and exponents of all kinds)."""
    import torch
    g = torch.Generator().manual_seed(seed)
    dt = getattr(torch, held)
    size = 1 if held == "float8_e4m3fn" else 2
    cache = tuple(torch.randint(0, 256, (pages, heads, page, d * size), generator=g, dtype=torch.uint8).view(dt) for _ in range(2))
    if size == 1:
        cache += tuple(torch.randint(0, 256, (pages, heads, page), generator=g, dtype=torch.uint8) for _ in range(2))
    return cache


def ints(x, pitch=None):
    import torch
    if pitch is None or not x:
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    whole = torch.full((len(x), pitch), 12345, dtype=torch.int32, device="cuda")
    whole[:, :len(x[0])] = torch.tensor(x, dtype=torch.int32)
    return whole[:, :len(x[0])]


def sequences(rng, pages, batch, width, page, share=0.5):
    """Consistent (users, table, lengths): rows that begin like the row before, and some empty ones."""
    users, table, lengths = [0] * pages, [], []
    free = list(range(pages))
    rng.shuffle(free)
    for b in range(batch):
        n = rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, width * page)])
        n = min(n, width * page)
        row = []
        if table and rng.random() < share:
            row = [p for p in table[-1][:-(-n // page)] if p >= 0]
        while len(row) < -(-n // page) and free:
            row.append(free.pop())
        n = min(n, len(row) * page)
        row = row[:-(-n // page)]
        for p in row:
            users[p] += 1
        table.append(row + [rng.choice([-1, -7])] * (width - len(row)))
        lengths.append(n)
    return users, table, lengths


SIZES = [(40, 1, 3, 16), (64, 7, 9, 16), (200, 33, 5, 64), (3000, 300, 11, 16), (9000, 2500, 3, 32), (17, 5, 1, 128), (5000, 700, 60, 16)]


@pytest.mark.parametrize("pages,batch,width,page", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
def test_fork(pages, batch, width, page, in_place):
    import torch
    import frisk_b200 as F
    rng = random.Random(pages + batch)
    cache = tuple(t.cuda() for t in new_cache(pages, 1, page, 64, "bfloat16"))
    users, table, lengths = sequences(rng, pages, batch, width, page)
    users[3] += 5  # (someone else holds a page too)
    for kind in ("any", "one", "gone", "same"):
        parents = [rng.randint(-1, batch - 1) if kind == "any" else {"one": rng.randrange(batch), "gone": -1, "same": b}[kind] for b in range(batch)]
        given = ints(users), ints(table, width + 3), ints(lengths)
        before = [t.clone() for t in given]
        got = F.cache_fork(cache, *given, ints(parents), out=given if in_place else None)
        F.cache_check()
        want = so.fork(users, table, lengths, parents, page)
        assert [t.tolist() for t in got] == list(want), kind
        if not in_place:
            assert all(torch.equal(a, b) for a, b in zip(given, before))


@pytest.mark.parametrize("pages,batch,width,page", SIZES)
@pytest.mark.parametrize("held", ["bfloat16", "float8_e4m3fn"])
@pytest.mark.parametrize("in_place", [False, True])
def test_grow(pages, batch, width, page, held, in_place):
    import frisk_b200 as F
    rng = random.Random(pages * 7 + batch)
    heads, d = (3, 64) if pages < 1000 else (1, 64)
    cpu = new_cache(pages, heads, page, d, held)
    for kind in ("one", "many", "too many", "none"):
        users, table, lengths = sequences(rng, pages, batch, width, page, 0.8)
        counts = [min(width * page - n, {"one": 1, "many": rng.randint(0, page + 3), "too many": rng.randint(0, width * page), "none": 0}[kind]) for n in lengths]
        if kind == "too many" and pages == 40:
            users = [max(n, 1) for n in users]  # (not one is free)
        starts = [2]
        for n in counts:
            starts.append(starts[-1] + n)
        given = ints(users), ints(table, width + 1), ints(starts), ints(lengths)
        cache = tuple(t.cuda() for t in cpu)
        out = (given[0], given[1], ints([-5] * batch)) if in_place else None
        got = F.cache_grow(cache, *given, out=out)
        F.cache_check()
        *want, copies = so.grow(users, table, starts, lengths, page)
        if not in_place:
            assert given[1].tolist() == table and given[0].tolist() == users
        assert [t.tolist() for t in got] == want, kind
        for come, go, keys in copies:
            for t in cpu:
                t.view(cpu[-1].dtype if held != "bfloat16" else t.dtype)[go, :, :keys] = t.view(cpu[-1].dtype if held != "bfloat16" else t.dtype)[come, :, :keys]
        assert same(cpu, cache), kind


@pytest.mark.parametrize("in_place", [False, True])
def test_many_pages(in_place):
    """More than a cluster copies, and free pages far behind the first."""
    import torch
    import frisk_b200 as F
    pages, batch, width, page = 300000, 500, 300, 16
    rng = random.Random(8)
    cache = F.paged_cache(pages, 1, page, 64, torch.float8_e4m3fn)
    users, table, lengths = sequences(rng, pages - 2000, batch, width - 1, page, 0.9)
    table = [r + [-1] for r in table]
    users = [max(n, 1) for n in users[:pages - 3000]] + users[pages - 3000:] + [0] * 2000  # (others have the first)
    parents = [rng.randint(-1, batch - 1) for _ in range(batch)]
    given = ints(users), ints(table), ints(lengths)
    got = F.cache_fork(cache, *given, ints(parents), out=given if in_place else None)
    want = so.fork(users, table, lengths, parents, page)
    assert [t.tolist() for t in got] == list(want)
    counts = [rng.randint(0, 20) for _ in range(batch)]
    counts = [min(n, width * page - m) for n, m in zip(counts, want[2])]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    got = F.cache_grow(cache, got[0], got[1], ints(starts), got[2], out=(got[0], got[1], ints([0] * batch)) if in_place else None)
    want = so.grow(*want[:2], starts, want[2], page)
    assert [t.tolist() for t in got] == list(want[:3])
    got = F.cache_compact(cache, got[0], got[1])
    want = so.compact(*want[:2])
    F.cache_check()
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and got[2].tolist() == [want[2]]


def test_grow_is_granted_in_order():
    """The first that lacks pages gets none, nor do those behind it, but for the ones that need none."""
    import frisk_b200 as F
    cache = tuple(t.cuda() for t in new_cache(6, 1, 16, 64, "float16"))
    users, table = [2, 1, 0, 0, 1, 1], [[0, -1, -1], [0, -1, -1], [1, -1, -1], [4, 5, -1]]
    lengths = [16, 10, 3, 32]
    # row 0 takes one page, row 1 a copy and one more (too many), row 2 has room, row 3 needs a page
    starts = [0, 1, 11, 13, 14]
    got = F.cache_grow(cache, ints(users), ints(table), ints(starts), ints(lengths))
    F.cache_check()
    assert got[2].tolist() == [1, 0, 2, 0]
    assert [t.tolist() for t in got] == list(so.grow(users, table, starts, lengths, 16)[:3])
    # three rows write into one page that no one else has: two take theirs, the last keeps it; if they cannot, it does not
    for free, want in ((2, [1, 1, 1]), (1, [1, 0, 0])):
        users = [3] + [0] * free + [1] * (5 - free)
        table = [[0, -1, -1]] * 3
        got = F.cache_grow(cache, ints(users), ints(table), ints([0, 1, 2, 3]), ints([4, 4, 4]))
        F.cache_check()
        assert got[2].tolist() == want
        assert [t.tolist() for t in got] == list(so.grow(users, table, [0, 1, 2, 3], [4, 4, 4], 16)[:3])


@pytest.mark.parametrize("batch,slots", [(3, 200), (4, 500), (40, 2500)])
def test_grow_over_many_shared_pages(batch, slots):
    """Rows that name the pages their new keys go to, all of them shared: the last row keeps what no one else has."""
    import torch
    import frisk_b200 as F
    others = [p % 7 == 0 for p in range(slots)]
    users, table, lengths = [batch + o for o in others] + [0] * batch * slots, [list(range(slots)) for _ in range(batch)], [3 + b % 12 for b in range(batch)]
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + slots * 16 - n)
    cache = F.paged_cache(len(users), 1, 16, 64, torch.float8_e4m3fn)
    got = F.cache_grow(cache, ints(users), ints(table), ints(starts), ints(lengths))
    F.cache_check()
    want = so.grow(users, table, starts, lengths, 16)
    assert [t.tolist() for t in got] == list(want[:3])
    # tables that name a page more often than is said: such pages are left
    few = [2 if p % 5 == 0 else n for p, n in enumerate(users[:slots])] + users[slots:]
    got = F.cache_grow(cache, ints(few), ints(table), ints(starts), ints(lengths))
    with pytest.raises(RuntimeError, match="table"):
        F.cache_check()
    left = torch.arange(0, slots, 5, device="cuda", dtype=torch.int32)
    assert torch.equal(got[1][:, ::5], left.expand(batch, -1)) and bool((got[0][left.long()] == 2).all())
    rest = torch.tensor([p for p in range(slots) if p % 5 and not others[p]], device="cuda")
    assert torch.equal(got[1][-1, rest], rest.int()) and bool((got[0][rest] == 1).all()) and bool((got[1][:-1, rest] >= slots).all())


@pytest.mark.parametrize("pages,page,held", [(1, 16, "bfloat16"), (33, 16, "float8_e4m3fn"), (700, 64, "float16"), (9001, 16, "float8_e4m3fn"), (257, 1024, "bfloat16")])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("full", [0.0, 0.3, 0.9, 1.0])
def test_compact(pages, page, held, in_place, full):
    import torch
    import frisk_b200 as F
    rng = random.Random(pages + int(10 * full))
    cpu = new_cache(pages, 1, page, 64, held)
    cache = tuple(t.cuda() for t in cpu)
    users = [rng.choice([1, 2, 5]) if rng.random() < full else 0 for _ in range(pages)]
    used = [p for p, n in enumerate(users) if n]
    width = 7
    table = [[rng.choice(used) if used and rng.random() < 0.8 else rng.choice([-1, -3]) for _ in range(width)] for _ in range(40)]
    given = ints(users), ints(table, 9)
    got = F.cache_compact(cache, *given, out=given + (ints([0]),) if in_place else None)
    F.cache_check()
    want_users, want_table, n, moves = so.compact(users, table)
    assert got[0].tolist() == want_users and got[1].tolist() == want_table and got[2].tolist() == [n]
    if moves:
        come, go = torch.tensor(list(moves)), torch.tensor(list(moves.values()))
        for t in cpu:
            raw = t.view(torch.uint8)
            raw[go] = raw[come]
    assert same(cpu, cache)


@pytest.mark.parametrize("heads,page,d,held", [(1, 16, 64, "float8_e4m3fn"), (3, 32, 128, "float8_e4m3fn"), (2, 16, 64, "float16"), (8, 64, 128, "bfloat16"), (5, 1024, 64, "bfloat16")])
@pytest.mark.parametrize("n", [0, 1, 23])
def test_copy(heads, page, d, held, n):
    import torch
    import frisk_b200 as F
    a, b = new_cache(31, heads, page, d, held, 1), new_cache(47, heads, page, d, held, 2)
    g = torch.Generator().manual_seed(3)
    source, target = torch.randint(0, 31, (n,), generator=g), torch.randperm(47, generator=g)[:n]
    ca, cb = tuple(t.cuda() for t in a), tuple(t.cuda() for t in b)
    assert F.cache_copy(ca, source.int().cuda(), target.int().cuda(), into=cb) is cb
    F.cache_check()
    want = [t.clone() for t in b]
    for x, y in zip(a, want):
        y.view(torch.uint8)[target] = x.view(torch.uint8)[source]
    assert same(want, cb) and same(a, ca)
    # within one cache
    source, target = torch.arange(min(n, 15)), torch.arange(min(n, 15)) + 15
    F.cache_copy(ca, source.int().cuda(), target.int().cuda())
    F.cache_check()
    for x in a:
        x.view(torch.uint8)[target] = x.view(torch.uint8)[source].clone()
    assert same(a, ca)


@pytest.mark.parametrize("counts,lengths,hkv,d,page", [([5], [0], 1, 64, 16), ([1, 7, 0, 24], [15, 16, 3, 40], 3, 64, 16), ([300, 33, 64], [1, 300, 127], 2, 128, 128),
                                                       ([2] * 70, list(range(70)), 8, 128, 32)])
@pytest.mark.parametrize("held", ["same", "float8_e4m3fn"])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_keep(counts, lengths, hkv, d, page, held, dtype):
    import torch
    import frisk_b200 as F
    batch = Batch(counts, lengths, hkv, 1, d, page, getattr(torch, dtype), None if held == "same" else torch.float8_e4m3fn, seed=len(counts))
    rng = random.Random(sum(counts))
    width = max(counts) + 2
    for kind in ("some", "all", "last", "none"):
        paths = []
        for n in counts:
            paths.append({"some": sorted(rng.sample(range(n), rng.randint(0, n))), "all": list(range(n)), "last": [n - 1] if n else [], "none": []}[kind])
        kept = ints([p + [rng.randint(-9, 999) for _ in range(width - len(p))] for p in paths], width + 5)
        batch.refresh()
        table, starts, lens = batch.plan
        for in_place in (True, False):
            mine = lens.clone()
            out = mine if in_place else None
            if not in_place:
                batch.refresh()
            got = F.cache_keep(batch.cache, table, starts, mine, kept, ints([len(p) for p in paths]), out=out)
            F.cache_check()
            assert got.tolist() == [n + len(p) for n, p in zip(lengths, paths)]
            assert in_place or torch.equal(mine, lens)
            want = [t.clone() for t in batch.cpu]
            for b, p in enumerate(paths):
                for i, at in enumerate(p):
                    come, go = lengths[b] + at, lengths[b] + i
                    for t in want:
                        raw = t.view(torch.uint8)
                        raw[int(batch.table_cpu[b, go // page]), :, go % page] = raw[int(batch.table_cpu[b, come // page]), :, come % page]
            assert same(want, batch.cache), (kind, in_place)


def test_what_tables_hold_out_of_range_is_left_out():
    """And said, without a memory access out of range."""
    import torch
    import frisk_b200 as F

    def says(call):
        got = call()
        with pytest.raises(RuntimeError, match="table"):
            F.cache_check()
        F.cache_check()
        return got

    cpu = new_cache(8, 2, 16, 64, "float8_e4m3fn")
    cache = tuple(t.cuda() for t in cpu)
    users, table, lengths = [1, 1, 1, 0, 0, 0, 0, 0], [[0, 1, -1], [2, -1, -1]], [20, 5]
    # parents; lengths: the row stays
    for parents, lens in (([0, 2], lengths), ([0, -2], lengths), ([0, 1 << 30], lengths)):
        got = says(lambda: F.cache_fork(cache, ints(users), ints(table), ints(lens), ints(parents)))
        assert [t.tolist() for t in got] == [users, table, lengths]
    for bad in (-1, 49, 1 << 30):
        got = says(lambda: F.cache_fork(cache, ints(users), ints(table), ints([20, bad]), ints([0, 1])))
        assert [t.tolist() for t in got] == [users, table, [20, bad]]
        got = says(lambda: F.cache_grow(cache, ints(users), ints(table), ints([0, 13, 14]), ints([20, bad])))
        assert got[2].tolist() == [13, 0] and got[1].tolist() == [[0, 1, 3], [2, -1, -1]] and got[0].tolist() == [1, 1, 1, 1, 0, 0, 0, 0]
    # starts
    for starts in ([0, 5, 4], [-3, 0, 1], [0, 1, 1 << 30], [0, -(1 << 31), 3]):
        got = says(lambda: F.cache_grow(cache, ints(users), ints(table), ints(starts), ints(lengths)))
        want = [0 if n < 0 or lo < 0 or n > 48 - m else n for n, lo, m in zip([b - a for a, b in zip(starts, starts[1:])], starts, lengths)]
        assert got[2].tolist() == want
    # pages
    bad = [[0, 99, -1], [2, 1 << 30, -1]]
    got = says(lambda: F.cache_fork(cache, ints(users), ints(bad), ints(lengths), ints([-1, -1])))
    assert got[0].tolist() == [0, 1, 0, 0, 0, 0, 0, 0] and got[1].tolist() == [[-1] * 3] * 2
    says(lambda: F.cache_grow(cache, ints(users), ints(bad), ints([0, 2, 3]), ints(lengths)))
    got = says(lambda: F.cache_compact(cache, ints([0, 1, 1, 0, 0, 0, 0, 0]), ints([[1, 8, 7], [2, 1 << 30, -1]])))
    assert got[1].tolist() == [[1, 8, 7], [0, 1 << 30, -1]] and got[2].tolist() == [2]
    cache = tuple(t.cuda() for t in cpu)
    for source, target in (([8], [0]), ([-1], [0]), ([0], [8]), ([0], [-1]), ([1 << 30], [1 << 30])):
        says(lambda: F.cache_copy(cache, ints(source), ints(target)))
    # accepted rows
    starts, lens = ints([0, 3, 5]), ints(lengths)
    for kept, counts in (([[0, 0, 1], [0, 1, 1]], [2, 0]), ([[1, 0, 1], [0, 1, 1]], [2, 0]), ([[0, 3, 1], [0, 1, 1]], [2, 0]), ([[-1, 2, 1], [0, 1, 1]], [2, 0]),
                         ([[0, 1, 2], [0, 1, 2]], [0, 3]), ([[0, 1, 2], [0, 1, 2]], [4, 0]), ([[0, 1, 2], [0, 1, 2]], [-1, 0])):
        got = says(lambda: F.cache_keep(cache, ints(table), starts, lens, ints(kept), ints(counts)))
        assert got.tolist() == lengths
    says(lambda: F.cache_keep(cache, ints([[0, 99, -1], [2, -1, -1]]), starts, lens, ints([[1, 2, 0], [0, 0, 0]]), ints([2, 0])))
    assert same(cpu, cache)


def test_offsets_beyond_32_bits():
    """Pages behind the first 2^32 bytes and 2^31 elements of keys."""
    import torch
    import frisk_b200 as F
    n, heads, page, d = 70000, 4, 64, 128
    cache = F.paged_cache(n, heads, page, d, torch.bfloat16)
    marks = torch.randn(2, 6, heads, page, d, device="cuda").bfloat16()
    at = [n - 1, n - 2, n - 3, 5, n - 4, n - 5]
    for t, m in zip(cache, marks):
        t.zero_()
        for i, p in enumerate(at[:4]):
            t[p] = m[i]
    # copied: the first backwards and the last forwards
    F.cache_copy(cache, ints([5, n - 1]), ints([n - 4, 6]))
    assert all(torch.equal(t[n - 4], m[3]) and torch.equal(t[6], m[0]) for t, m in zip(cache, marks))
    # a shared last page is written: its keys go to the only free page
    users = torch.ones(n, dtype=torch.int32, device="cuda")
    users[n - 2], users[n - 5] = 2, 0
    table = ints([[n - 2, -1], [n - 2, -1]])
    users, table, granted = F.cache_grow(cache, users, table, ints([0, 1, 1]), ints([50, 50]))
    assert table.tolist() == [[n - 5, -1], [n - 2, -1]] and granted.tolist() == [1, 0] and int(users[n - 5]) == 1
    assert all(torch.equal(t[n - 5, :, :50], m[1, :, :50]) for t, m in zip(cache, marks))
    # accepted rows move within the page, and over its end
    got = F.cache_keep(cache, ints([[n - 3, n - 1]]), ints([0, 8]), ints([62]), ints([[0, 3, 7]]), ints([3]))
    assert got.tolist() == [65]
    for t, m in zip(cache, marks):
        assert torch.equal(t[n - 3, :, :63], m[2, :, :63]) and torch.equal(t[n - 3, :, 63], m[0, :, 1])
        assert torch.equal(t[n - 1, :, 0], m[0, :, 5]) and torch.equal(t[n - 1, :, 1:], m[0, :, 1:])
    # the last page comes to the front
    users = torch.zeros(n, dtype=torch.int32, device="cuda")
    users[n - 2] = 3
    users, table, used = F.cache_compact(cache, users, ints([[n - 2, -1]]))
    F.cache_check()
    assert table.tolist() == [[0, -1]] and used.tolist() == [1] and int(users[0]) == 3 and int(users.sum()) == 3
    assert all(torch.equal(t[0], m[1]) for t, m in zip(cache, marks))


def test_refusals():
    import torch
    import frisk_b200 as F
    cache = F.paged_cache(8, 2, 16, 64, torch.bfloat16)
    users, table, lengths = F.page_tables(cache, 2, 3)
    i, starts = ints([0, 1]), ints([0, 1, 2])
    for call in (lambda: F.cache_fork(cache, users[:7], table, lengths, i), lambda: F.cache_fork(cache, users.long(), table, lengths, i),
                 lambda: F.cache_fork(cache, users, table, lengths, ints([0])), lambda: F.cache_fork(cache, users, table.t(), lengths, i),
                 lambda: F.cache_fork(cache, users, table, lengths, i, out=(users, table)), lambda: F.cache_fork(cache, users, table, lengths, i, out=(users, table[:, :2], lengths)),
                 lambda: F.cache_fork(cache, users, table, lengths, i, out=(users, table, i)),               # a result in the place of another input
                 lambda: F.cache_fork(cache, users, table, lengths, i, out=(users, table, users[:2])),       # of another result
                 lambda: F.cache_fork(cache, users, table, lengths, i.cpu()),
                 lambda: F.cache_grow(cache, users, table, i, lengths), lambda: F.cache_grow(cache, users, table, starts, lengths, out=(users, table, lengths)),
                 lambda: F.cache_compact(cache, users, table, out=(users, table, users[:1])), lambda: F.cache_compact(cache[:1], users, table),
                 lambda: F.cache_compact((cache[0], cache[0]), users, table),                                  # keys and values in one place
                 lambda: F.cache_copy(cache, i, ints([0])), lambda: F.cache_copy(cache, i, i, into=F.paged_cache(8, 2, 32, 64, torch.bfloat16)),
                 lambda: F.cache_copy(cache, i, i, into=F.paged_cache(8, 2, 16, 64, torch.float16)), lambda: F.cache_copy(cache, i, i, into=(cache[1], cache[0])),
                 lambda: F.cache_copy(cache, i.long(), i.long()), lambda: F.cache_keep(cache, table, starts, lengths, table[:1], i),
                 lambda: F.cache_keep(cache, table, starts, lengths, table, i, out=i), lambda: F.cache_keep(cache, table, starts, lengths, table, ints([0])),
                 lambda: F.cache_keep(cache, table, starts, lengths, table, starts)):
        with pytest.raises(ValueError):
            call()
    # nothing to do
    empty = F.page_tables(cache, 0, 3)
    none = ints([])
    assert [t.shape[0] for t in F.cache_fork(cache, *empty, none)] == [8, 0, 0]
    assert [t.shape[0] for t in F.cache_grow(cache, empty[0], empty[1], ints([0]), empty[2])] == [8, 0, 0]
    assert F.cache_keep(cache, empty[1], ints([0]), empty[2], empty[1], none).shape == (0,)
    users, table, used = F.cache_compact(cache, *empty[:2])
    assert used.tolist() == [0]
    wide = F.page_tables(cache, 2, 0)
    assert F.cache_grow(cache, wide[0], wide[1], ints([0, 0, 0]), wide[2])[2].tolist() == [0, 0]
    F.cache_check()


def test_a_stream_of_its_own_and_a_graph():
    """Results of a captured step, in place, replayed for other contents, are those of calls made one by one."""
    import torch
    import frisk_b200 as F
    rng = random.Random(4)
    pages, batch, width, page = 300, 20, 12, 16
    cache = tuple(t.cuda() for t in new_cache(pages, 2, page, 64, "bfloat16"))
    users, table, lengths = (ints(x) for x in sequences(rng, pages, batch, width - 2, page))
    table = torch.nn.functional.pad(table, (0, 2), value=-1).contiguous()
    starts, parents, granted = ints(list(range(batch + 1))), ints([0] * batch), ints([0] * batch)
    side = torch.cuda.Stream()

    def step():
        F.cache_fork(cache, users, table, lengths, parents, out=(users, table, lengths))
        F.cache_grow(cache, users, table, starts, lengths, out=(users, table, granted))
        lengths.add_(granted)

    start = [t.clone() for t in (users, table, lengths) + cache]
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        step()
    torch.cuda.synchronize()
    for t, s in zip((users, table, lengths) + cache, start):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, s in zip((users, table, lengths) + cache, start):
        t.copy_(s)
    host = [t.tolist() for t in start[:3]]
    for turn in range(4):
        now = [rng.randint(-1, batch - 1) for _ in range(batch)]
        parents.copy_(ints(now))
        graph.replay()
        F.cache_check()
        host = list(so.fork(*host, now, page))
        u, t, g, _ = so.grow(host[0], host[1], list(range(batch + 1)), host[2], page)
        host = [u, t, [n + m for n, m in zip(host[2], g)]]
        assert [x.tolist() for x in (users, table, lengths)] == host and granted.tolist() == g
    # the stream can be named
    a = F.cache_fork(cache, users, table, lengths, parents, stream=side)
    b = F.cache_grow(cache, a[0], a[1], starts, a[2], stream=side)
    side.synchronize()
    want = so.fork(*host, now, page)
    assert [x.tolist() for x in a] == list(want)
    assert [x.tolist() for x in b] == list(so.grow(want[0], want[1], list(range(batch + 1)), want[2], page)[:3])
