"""Tables of shared pages that contradict their users: what `cache_grow` may hand out, and what it says."""
import pytest

pytestmark = pytest.mark.gpu


def ints(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def grown(cache, users, table, starts, lengths, in_place=False):
    """The call's results as lists, and whether `cache_check` raises behind it."""
    import frisk_b200 as F
    users, table = ints(users), ints(table)
    got = F.cache_grow(cache, users, table, ints(starts), ints(lengths), out=(users, table, ints([0] * len(lengths))) if in_place else None)
    said = False
    try:
        F.cache_check()
    except RuntimeError as e:
        said = "table" in str(e)
    F.cache_check()
    return [t.tolist() for t in got], said


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bad", [0, -3])
def test_a_page_without_users_is_not_written(bad, in_place):
    """A row names a page that is said to be free: it is granted nothing and nobody else gets the page; the others get theirs as if it asked for nothing."""
    import torch
    import frisk_b200 as F
    cache = F.paged_cache(8, 1, 16, 64, torch.bfloat16)
    # row 0: page 0 and a new one; row 1: page 1 (no users) and a new one; row 2: a new one
    users, table = [1, bad, 1, 0, 0, 0, 0, 0], [[0, -1, -1], [1, -1, -1], [2, -1, -1]]
    got, said = grown(cache, users, table, [0, 10, 30, 34], [10, 10, 14], in_place)
    assert said and got == [[1, bad, 1, 1, 1, 0, 0, 0], [[0, 3, -1], [1, -1, -1], [2, 4, -1]], [10, 0, 4]]
    # the page behind the last key (a row that holds pages ahead): the same, the first page, which others have, is left too
    users, table = [2, 1, bad, 0, 0, 0, 0, 0], [[0, 2, -1], [0, 1, -1]]
    got, said = grown(cache, users, table, [0, 12, 15], [10, 12], in_place)
    assert said and got == [[1, 1, bad, 1, 0, 0, 0, 0], [[0, 2, -1], [3, 1, -1]], [0, 3]]


@pytest.mark.parametrize("in_place", [False, True])
def test_a_page_of_one_user_that_two_rows_name_is_said(in_place):
    import torch
    import frisk_b200 as F
    cache = F.paged_cache(8, 1, 16, 64, torch.bfloat16)
    users, table, lengths = [1, 1, 0, 0, 0, 0, 0, 0], [[0, -1], [1, -1], [0, -1]], [4, 5, 6]
    got, said = grown(cache, users, table, [0, 1, 2, 3], lengths, in_place)
    assert said and got == [users, table, [1, 1, 1]]
    # twice in one row
    got, said = grown(cache, [1, 1, 0, 0, 0, 0, 0, 0], [[0, 0], [1, -1]], [0, 15, 16], [4, 5], in_place)
    assert said and got[1] == [[0, 0], [1, -1]]
    # only rows that write are looked at; and pages of one user each are nothing to say
    for starts in ([0, 1, 2, 2], [0, 0, 1, 2]):
        got, said = grown(cache, users, table, starts, lengths, in_place)
        assert not said and got[:2] == [users, table]


@pytest.mark.parametrize("batch,slots", [(6, 40), (60, 100)])
def test_many_rows_of_pages_that_are_said_wrong(batch, slots):
    """Fewer slots than shared memory holds, and more."""
    import torch
    import frisk_b200 as F
    pages = 2 * batch * slots + 50
    cache = F.paged_cache(pages, 1, 16, 64, torch.float8_e4m3fn)
    table = [list(range(b * slots, (b + 1) * slots - 2)) + [-1, -1] for b in range(batch)]
    users = [0] * pages
    for row in table:
        for p in row[:-2]:
            users[p] = 1
    starts = [n * (slots * 16 - 5) for n in range(batch + 1)]
    lengths = [5] * batch
    got, said = grown(cache, users, table, starts, lengths)
    fresh = [p for p, n in enumerate(users) if n == 0]
    want = [row[:-2] + fresh[2 * b:2 * b + 2] for b, row in enumerate(table)]
    assert not said and got[1] == want and got[2] == [slots * 16 - 5] * batch
    # one page of row 2 has no users, and one of row 3 is row 4's too
    wrong = list(users)
    wrong[table[2][7]] = 0
    table[3][9] = table[4][9]
    got, said = grown(cache, wrong, table, starts, lengths)
    keeps = [p for p, n in enumerate(wrong) if n == 0 and p != table[2][7]]
    rows = [row[:-2] for row in table]
    at = 0
    for b in range(batch):
        if b == 2:
            rows[b] = rows[b] + [-1, -1]
        else:
            rows[b] = rows[b] + keeps[at:at + 2]
            at += 2
    assert said and got[1] == rows and got[2] == [0 if b == 2 else slots * 16 - 5 for b in range(batch)] and got[0][table[2][7]] == 0
