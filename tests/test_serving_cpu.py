"""What the entries for pages, drafts and adapters refuse before anything is launched, and the definitions they are tested against."""
import ctypes

import pytest
import torch

import frisk_b200 as F
from frisk_b200 import capi
from oracle import serving_oracle as so


def _cache(**change):
    d = dict(pages=8, page=16, heads=2, D=64, dtype=capi.BF16, batch=2, table_width=4, table_stride=4, rows=2 ** 31 - 1, k=1 << 30, v=2 << 30,
             k_exponent=None, v_exponent=None, table=3 << 20, starts=4 << 20, lengths=5 << 20)
    d.update(change)
    return capi.CacheDesc(**d)


def test_workspace_sizes_say_what_is_refused():
    size = capi.cache_pages_workspace_bytes
    for which in (capi.PAGES_FORK, capi.PAGES_GROW, capi.PAGES_COMPACT):
        assert size(_cache(batch=4000, table_width=100, table_stride=100), which) > 0
        assert (size(_cache(), which) > 0) == (which != capi.PAGES_FORK)  # (small tables are forked without)
        for change in (dict(page=8), dict(page=24), dict(D=96), dict(heads=0), dict(pages=0), dict(batch=-1), dict(table_width=-1), dict(table_stride=3),
                       dict(dtype=capi.F32), dict(pages=1 << 40), dict(batch=1 << 20, table_width=1 << 12, table_stride=1 << 12),
                       dict(table_width=1 << 28, table_stride=1 << 28)):
            assert size(_cache(**change), which) == 0, (which, change)
    assert size(_cache(), 3) == 0 and size(_cache(), -1) == 0


def test_adapters_beyond_the_limits_need_no_workspace():
    def size(rows, n, rank=8):
        return capi.adapter_workspace_bytes(capi.AdapterDesc(rows, 64, n, 64, 64, 64 * rank, rank, rank * n, n, n, rank, 1, 1, capi.BF16, capi.BF16))

    assert size(1 << 26, 64) >= (1 << 26) * 8 * 2 * 2 and size((1 << 26) + 1, 64) == 0
    assert size(512, 1 << 28) > 0 and size(512, (1 << 28) + 8) == 0 and size(512, 64, 12) == 0 and size(512, 64, 136) == 0


def test_null_contexts_are_refused():
    lib = capi.load()
    t = capi.PageTables(1 << 20, 1 << 21, 1 << 22, 1 << 23, 4)
    assert lib.frisk_b200_cache_fork(None, _cache(), t, 1 << 24, 1 << 25, 1 << 20, None) == -7
    assert lib.frisk_b200_cache_grow(None, _cache(), t, 1 << 25, 1 << 20, None) == -7
    assert lib.frisk_b200_cache_compact(None, _cache(), t, 1 << 25, 1 << 20, None) == -7
    assert lib.frisk_b200_cache_copy(None, _cache(), _cache(), 1 << 20, 1 << 21, 1, None) == -7
    assert lib.frisk_b200_cache_keep(None, _cache(), 1 << 20, 4, 4, 1 << 21, 1 << 22, None) == -7
    assert lib.frisk_b200_draft_verify(None, capi.VerifyDesc(1, 8, 0, 1, 1, 8, 0, 0), *[1 << 20] * 10, None) == -7
    assert lib.frisk_b200_adapter_gemm(None, capi.AdapterDesc(), *[1 << 20] * 9, 1 << 20, None) == -7
    assert ctypes.sizeof(capi.PageTables) == 40 and ctypes.sizeof(capi.VerifyDesc) == 48 and ctypes.sizeof(capi.AdapterDesc) == 104


def test_what_is_not_on_a_device_is_refused():
    cache = F.paged_cache(4, 2, 16, 64, torch.float16, device="cpu")
    users, table, lengths = F.page_tables(cache, 2, 3)
    assert users.tolist() == [0] * 4 and table.tolist() == [[-1] * 3] * 2 and lengths.tolist() == [0, 0]
    starts, i = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    f, x = torch.zeros(2), torch.zeros(2, 8, dtype=torch.float16)
    a, b = torch.zeros(1, 8, 8, dtype=torch.float16), torch.zeros(1, 8, 8, dtype=torch.float16)
    for call in (lambda: F.cache_fork(cache, users, table, lengths, i), lambda: F.cache_grow(cache, users, table, starts, lengths),
                 lambda: F.cache_compact(cache, users, table), lambda: F.cache_copy(cache, i, i), lambda: F.cache_keep(cache, table, starts, lengths, table, i),
                 lambda: F.draft_verify(i.long(), None, starts, torch.zeros(2, 5), None, f, f, max_new=2), lambda: F.adapter_gemm(x, a, b, x, starts, i)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        F.page_tables(cache, -1, 2)


def test_the_definitions():
    """Small cases worked out by hand."""
    # pages 0..3 of one sequence of 20 keys; two more rows take it over, the second sequence ends
    users, table, lens = so.fork([1, 1, 1, 0], [[0, 1, -1], [2, -1, -1], [-1] * 3], [20, 3, 0], [0, -1, 0], 16)
    assert users == [2, 2, 0, 0] and table == [[0, 1, -1], [-1] * 3, [0, 1, -1]] and lens == [20, 0, 20]
    # both write: the first takes a page and the four keys, the last keeps what it has
    users, table, granted, copies = so.grow(users, table, [0, 1, 1, 2], lens, 16)
    assert users == [2, 1, 1, 0] and table == [[0, 2, -1], [-1] * 3, [0, 1, -1]] and granted == [1, 0, 1] and copies == [(1, 2, 4)]
    # thirteen more keys for the first, twelve for the last: one page is left
    users, table, granted, copies = so.grow(users, table, [0, 13, 13, 25], [20, 0, 20], 16)
    assert granted == [13, 0, 12] and users == [2, 1, 1, 1] and table[0] == [0, 2, 3] and copies == []
    assert so.compact([0, 1, 0, 2], [[3, -1], [1, 3]]) == ([2, 1, 0, 0], [[0, -1], [1, 0]], 2, {3: 0})
    # a chain: 0.5 of the first token stands for u < 0.5; what is left of the second is its own row without it
    p = torch.tensor([[0.5, 0.25, 0.25], [0.0, 0.5, 0.5], [1.0, 0.0, 0.0]])
    assert so.verify([9, 0, 1], None, [0, 3], p, None, [0.0, 0.49, 0.5], [0.0], 4) == ([[0, 1, -1, -1]], [2], [2])
    assert so.verify([9, 0, 1], None, [0, 3], p, None, [0.0, 0.49, 0.49], [0.99], 4) == ([[0, 1, 2, -1]], [3], [0])
    assert so.verify([9, 0, 1], None, [0, 3], p, None, [0.0, 0.5, 0.0], [0.5], 4) == ([[0, -1, -1, -1]], [1], [2])
    # a draft that never draws the last token: rejected, it is all that is left
    q = torch.tensor([[0.75, 0.25, 0.0]] * 3)
    assert so.verify([9, 0, 1], None, [0, 3], p, q, [0.0, 0.7, 0.0], [0.5], 3) == ([[0, -1, -1]], [1], [2])


def test_tokens_are_distributed_as_the_targets():
    """Two children drawn from the draft, whatever it is: the first token behind the root has the target's distribution, to six deviations."""
    g = torch.Generator().manual_seed(5)
    n, p, q = 20000, torch.tensor([0.5, 0.2, 0.3, 0.0]), torch.tensor([0.1, 0.6, 0.1, 0.2])
    drawn = torch.multinomial(q, 2 * n, replacement=True, generator=g).view(n, 2).tolist()
    accept, sample = torch.rand(n, 2, generator=g).tolist(), torch.rand(n, generator=g).tolist()
    rows, drafts = p.repeat(3, 1), q.repeat(3, 1)
    seen = [0] * 4
    for d, u, s in zip(drawn, accept, sample):
        kept, counts, token = so.verify([0] + d, [-1, 0, 0], [0, 3], rows, drafts, [0.0] + u, [s], 3)
        seen[d[kept[0][1] - 1] if counts[0] > 1 else token[0]] += 1
    for have, want in zip(seen, p.tolist()):
        assert abs(have / n - want) <= 6 * (want * (1 - want) / n) ** 0.5
