"""Results of the cache's operators in columns of a shared buffer, heads before rows, and what is refused."""
import pytest
import torch

import frisk_b200 as F
from tests.test_cache_gpu import Batch

pytestmark = pytest.mark.gpu


def batch(held=None):
    return Batch([5, 30, 1], [70, 3, 200], 2, 4, 64, 16, torch.bfloat16, held, 31)


@pytest.mark.parametrize("e4m3", [False, True])
def test_rows_are_read_into_one_buffer(e4m3):
    b = batch(torch.float8_e4m3fn if e4m3 else None)
    want = F.cache_read(b.cache, *b.plan, b.rows, dtype=torch.bfloat16)
    n, h, d = b.rows, 2, 64
    whole = torch.full((n, h, 3, d), 5.0, dtype=torch.bfloat16, device="cuda")  # queries, keys and values side by side in each head
    F.cache_read(b.cache, *b.plan, n, out=(whole[:, :, 1], whole[:, :, 2]))
    assert torch.equal(whole[:, :, 1], want[0]) and torch.equal(whole[:, :, 2], want[1]) and bool((whole[:, :, 0] == 5).all())
    columns = torch.full((n, 5, d), 5.0, dtype=torch.bfloat16, device="cuda")
    F.cache_read(b.cache, *b.plan, n, out=(columns[:, :2], columns[:, 3:]))
    assert torch.equal(columns[:, :2], want[0]) and torch.equal(columns[:, 3:], want[1]) and bool((columns[:, 2] == 5).all())
    heads = torch.full((2, h, n, d), 5.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2)  # heads before rows
    F.cache_read(b.cache, *b.plan, n, out=(heads[0], heads[1]))
    assert torch.equal(heads[0], want[0]) and torch.equal(heads[1], want[1])
    F.cache_check()
    for k, v in ((columns[:, :2], columns[:, 1:3]), (columns[:, :2], columns[:, :2]), (whole[:, :, 1], whole.view(n, 3 * h, d)[:, 1:3])):
        with pytest.raises(ValueError):
            F.cache_read(b.cache, *b.plan, n, out=(k, v))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("tile_rows", [16, 128, 256])
def test_results_beside_queries(e4m3, tile_rows):
    b = batch(torch.float8_e4m3fn if e4m3 else None)
    n, h, d = b.q.shape
    want = F.cache_attention(b.cache, b.q, *b.plan, tile_rows=tile_rows)
    sides = torch.full((n, h, 2, d), 5.0, dtype=b.dtype, device="cuda")
    columns = torch.full((n, 2 * h, d), 5.0, dtype=b.dtype, device="cuda")
    for q, out in ((sides[:, :, 0], sides[:, :, 1]), (columns[:, :h], columns[:, h:]), (b.q, torch.empty(h, n, d, dtype=b.dtype, device="cuda").transpose(0, 1))):
        q.copy_(b.q)
        F.cache_attention(b.cache, q, *b.plan, tile_rows=tile_rows, out=out)
        assert torch.equal(out, want) and torch.equal(q, b.q)
    F.cache_check()
    for q, out in ((columns[:, :h], columns[:, 1:h + 1]), (sides[:, :, 0], sides[:, :, 0]), (b.q, want[:, :1].expand(n, h, d)),
                   (b.q, torch.empty(1, 1, d, dtype=b.dtype, device="cuda").expand(n, h, d))):
        with pytest.raises(ValueError):
            F.cache_attention(b.cache, q, *b.plan, tile_rows=tile_rows, out=out)
