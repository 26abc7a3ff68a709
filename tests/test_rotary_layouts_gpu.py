"""Rotary positions in place and beside other tensors: which layouts are taken, and that nothing else is written."""
import pytest
import torch

import frisk_b200 as F

pytestmark = pytest.mark.gpu

N, H, D = 33, 3, 64


def places(t):
    """The elements of ``t`` in its buffer."""
    at = torch.full(t.shape, t.storage_offset(), dtype=torch.int64)
    for i, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s).view([-1 if j == i else 1 for j in range(t.dim())])
    return at.flatten()


def buffer(seed=1):
    return torch.randn(40 * 3 * 8 * 80, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


# (offset, shape, strides) of queries and of keys in one buffer
ROWS = {
    "columns": ((0, (N, H, D), (1024, D, 1)), (H * D, (N, 2, D), (1024, D, 1))),
    "queries, keys and values side by side in each head": ((0, (N, H, D), (H * 3 * D, 3 * D, 1)), (D, (N, H, D), (H * 3 * D, 3 * D, 1))),
    "the same, fewer heads of keys": ((0, (N, H, D), (H * 3 * D, 3 * D, 1)), (2 * D, (N, 1, D), (H * 3 * D, D, 1))),
    "the same, halves of heads": ((D // 2, (N, H, D // 2), (H * 3 * D, 3 * D, 1)), (D + 8, (N, H, D // 2), (H * 3 * D, 3 * D, 1))),
    "heads before rows": ((0, (N, H, D), (D, N * D, 1)), (H * N * D, (N, 2, D), (D, N * D, 1))),
    "heads before rows, side by side": ((0, (N, H, D), (2 * D, N * 2 * D, 1)), (D, (N, H, D), (2 * D, N * 2 * D, 1))),
    "rows of two tensors in turn": ((0, (N, H, D), (2 * H * D, D, 1)), (H * D, (N, H, D), (2 * H * D, D, 1))),
}


@pytest.mark.parametrize("name", ROWS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place(name, interleaved):
    buf = buffer()
    q, k = (torch.as_strided(buf, shape, strides, offset) for offset, shape, strides in ROWS[name])
    used = torch.cat((places(q), places(k)))
    assert len(used.unique()) == len(used)
    d = q.shape[2]
    positions, (f, _) = torch.arange(N, device="cuda") * 1001, F.rotary_frequencies(d)
    before = buf.clone()
    want = F.rotary(q.contiguous(), k.contiguous(), positions, f, interleaved=interleaved)
    F.rotary(q, k, positions, f, interleaved=interleaved, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    rest = torch.ones(len(buf), dtype=torch.bool)
    rest[used] = False
    assert torch.equal(buf.cpu()[rest], before.cpu()[rest])


def test_queries_into_the_places_of_values():
    """Not in place, but between the inputs of one buffer: heads of (queries, results, keys)."""
    buf = buffer(2).narrow(0, 0, N * H * 3 * D).view(N, H, 3, D)
    q, out, k = buf.unbind(2)
    positions, (f, _) = torch.arange(N, device="cuda"), F.rotary_frequencies(D)
    want = F.rotary(q.contiguous(), k.contiguous(), positions, f)
    F.rotary(q, k, positions, f, out=(out, k))
    assert torch.equal(out, want[0]) and torch.equal(k, want[1])


OVERLAPPING = [
    ((0, (N, H, D), (H * 3 * D, 3 * D, 1)), (D - 8, (N, H, D), (H * 3 * D, 3 * D, 1))),
    ((0, (N, H, D), (H * 3 * D, 3 * D, 1)), (D, (N, H, D), (H * 3 * D, D, 1))),
    ((0, (N, H, D), (D, N * D, 1)), ((H - 1) * N * D + 64, (N, H, D), (D, N * D, 1))),
    ((0, (N, H, D), (1024, D, 1)), ((H - 1) * D, (N, 2, D), (1024, D, 1))),
    ((0, (N, H, D), (1024, D, 1)), (H * D, (N, 2, D), (1024 + D, D, 1))),
]


@pytest.mark.parametrize("queries,keys", OVERLAPPING)
def test_results_over_other_tensors_are_refused(queries, keys):
    buf = buffer()
    q, k = (torch.as_strided(buf, shape, strides, offset) for offset, shape, strides in (queries, keys))
    used = torch.cat((places(q), places(k)))
    assert len(used.unique()) < len(used)
    positions, (f, _) = torch.arange(N, device="cuda"), F.rotary_frequencies(D)
    before = buf.clone()
    for out in ((q, k), (q, torch.empty(k.shape, dtype=k.dtype, device="cuda")), (torch.empty(q.shape, dtype=q.dtype, device="cuda"), k)):
        with pytest.raises(ValueError):
            F.rotary(q, k, positions, f, out=out)
    for shape, strides in (((N, H, D), (D, D, 1)), ((N, H, D), (D // 2, N * D, 1)), ((N, H, D), (H * D - 8, D, 1))):  # over itself
        own = torch.as_strided(buf, shape, strides, 0)
        with pytest.raises(ValueError):
            F.rotary(own, None, positions, f, out=(own, None))
    assert torch.equal(buf, before)
