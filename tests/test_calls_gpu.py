"""The native form of the serving operators' calls (csrc/calls.cpp): the same results as the Python functions', and None for all that is not usual."""
import pytest

from tests.test_adapters_gpu import Requests
from tests.test_drafts_gpu import Drafts
from tests.test_pages_gpu import ints, new_cache

pytestmark = pytest.mark.gpu


@pytest.fixture
def calls():
    import torch
    import frisk_b200 as F
    from frisk_b200 import calls
    calls.context_for(0)
    if not calls.path(torch.__version__).exists():
        pytest.skip("built without native calls")
    return calls


def arguments():
    """Of each operator: the function, its arguments, the native one and its arguments."""
    import torch
    import frisk_b200 as F
    from frisk_b200 import calls, capi
    d = Drafts([3, 5, 1], 300)
    i32 = dict(dtype=torch.int32, device="cuda")
    verify = [d.tokens.cuda(), torch.tensor(d.parents, **i32), torch.tensor(d.starts, **i32), d.target.cuda(), d.draft.cuda(), d.accept.cuda(), d.sample.cuda()]
    r = Requests([3, 1, 2], 64, 40, 16, 2, seed=1)
    x, a, b, c = (t.cuda()[..., s] for t, s in zip(r.whole, r.cut))
    adapters = [x, a, b, c, torch.tensor(r.starts, **i32), torch.tensor([1, -1, 0], **i32), r.scales.cuda()]
    cache = tuple(t.cuda() for t in new_cache(9, 2, 16, 64, "float8_e4m3fn"))
    users, table, lengths, starts = ints([1, 1, 2, 0, 0, 0, 0, 0, 0]), ints([[0, 2, -1], [1, 2, -1]], 5), ints([20, 25]), ints([0, 2, 4])
    other = tuple(t.cuda() for t in new_cache(9, 2, 16, 64, "float8_e4m3fn", 1))
    kept, counts = ints([[0, 1], [1, 1]]), ints([2, 1])
    torch.manual_seed(6)
    rows = torch.randn(4, 4, 64, device="cuda").bfloat16()
    fork, grow, compact = capi.PAGES_FORK, capi.PAGES_GROW, capi.PAGES_COMPACT
    return {
        "verify": (lambda *v: F.draft_verify(*v, max_new=6), verify, calls.verify, verify + [6]),
        "adapters": (lambda *v: F.adapter_gemm(*v[:6], scales=v[6]), adapters, calls.adapters, adapters),
        "fork": (F.cache_fork, [cache, users, table, lengths, ints([1, 0])], calls.change, [fork, cache, users, table, None, lengths, ints([1, 0])]),
        "grow": (F.cache_grow, [cache, users, table, starts, lengths], calls.change, [grow, cache, users, table, starts, lengths, None]),
        "compact": (F.cache_compact, [cache, users, table], calls.change, [compact, cache, users, table, None, None, None]),
        "keep": (F.cache_keep, [cache, table, starts, lengths, kept, counts], calls.keep, [cache, table, starts, lengths, kept, counts]),
        "copy": (lambda a, b, c, d: F.cache_copy(a, b, c, into=d), [cache, ints([1, 0]), ints([4, 8]), other], calls.copy, [cache, ints([1, 0]), ints([4, 8]), other]),
        "write": (F.cache_write, [cache, rows[:, :2], rows[:, 2:], table, starts, lengths], calls.write, [cache, rows[:, :2], rows[:, 2:], table, starts, lengths]),
    }


def flat(x):
    import torch
    return [t.cpu().view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.cpu() for t in ((x,) if isinstance(x, torch.Tensor) else x)]


@pytest.mark.parametrize("name", ["verify", "adapters", "fork", "grow", "compact", "keep", "copy", "write"])
def test_the_same_as_python(calls, name, monkeypatch):
    import torch
    import frisk_b200 as F
    function, args, native, native_args = arguments()[name]
    given = native(*native_args)
    assert given is not None and type(given) is not int
    first = flat(function(*args))
    for other in ("verify", "change", "keep", "copy", "adapters", "write"):
        monkeypatch.setattr(calls, other, lambda *_: None)
    function, args, _, _ = arguments()[name]  # (what a call changed in place is as it was)
    second = flat(function(*args))
    F.cache_check()
    assert all(torch.equal(a, b) for a, b in zip(first, second)) and len(first) == len(second)
    if given is not True:
        assert all(torch.equal(a, b) for a, b in zip(flat(given), first))


@pytest.mark.parametrize("name", ["verify", "adapters", "fork", "grow", "compact", "keep", "copy", "write"])
def test_what_is_unusual_is_left_to_python(calls, name):
    import torch

    class Other(torch.Tensor):
        pass

    _, _, native, args = arguments()[name]
    assert native() is None and native(*args[:-1]) is None and native(*args, None) is None
    for i, one in enumerate(args):
        tensors = one if isinstance(one, tuple) else (one,)
        for j, t in enumerate(tensors):
            if not isinstance(t, torch.Tensor):
                continue
            # another type of object, of element, of device, of class; another shape; elements that are no neighbours
            spread = torch.stack((t, t), -1)[..., 0] if t.dtype != torch.float8_e4m3fn else t.transpose(0, 1)
            for bad in (3, "x", t.cpu(), t.to(torch.float64), t.as_subclass(Other), t[None], spread):
                put = tuple(bad if k == j else x for k, x in enumerate(one)) if isinstance(one, tuple) else bad
                assert native(*args[:i], put, *args[i + 1:]) is None, (i, j)
        if isinstance(one, tuple):
            for bad in (list(one), one[:1], one + one[:1], ()):
                assert native(*args[:i], bad, *args[i + 1:]) is None
    for i, one in enumerate(args):
        if type(one) is int:
            for bad in (None, 1.0, 1 << 70, -1 if name == "verify" else "0"):
                assert native(*args[:i], bad, *args[i + 1:]) is None
    torch.cuda.synchronize()


def test_errors_of_the_library_are_raised(calls):
    import torch
    import frisk_b200 as F
    _, args, native, native_args = arguments()["adapters"]
    odd = torch.zeros(6, 65, device="cuda").bfloat16()[:, 1:]  # rows that do not begin on 16 bytes
    assert native(odd, *native_args[1:]) == -3
    with pytest.raises(ValueError, match="aligned"):
        F.adapter_gemm(odd, *args[1:6])
    cache = F.paged_cache(8, 2, 16, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="overlaps"):
        F.cache_compact((cache[0], cache[0]), *F.page_tables(cache, 2, 3)[:2])


def test_on_the_current_stream(calls):
    """And in a graph: results belong to the stream that is current."""
    import torch
    import frisk_b200 as F
    function, args, _, _ = arguments()["adapters"]
    want = function(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = function(*args)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = function(*args)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_results_of_one_call_are_tensors_of_their_own(calls):
    """They share an allocation: each is dense, on its own bytes, and may be changed, kept and passed on by itself."""
    import torch
    import frisk_b200 as F
    made = arguments()
    for name in ("verify", "fork", "grow", "compact"):
        function, args, _, _ = made[name]
        first, second = function(*args), function(*args)
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in first + second)
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
        for i, (t, want) in enumerate(zip(first, second)):
            assert t.is_contiguous() and t.device == args[1].device and not t.requires_grad and t.shape == want.shape and t.dtype == want.dtype
            before = [u.clone() for u in first]
            t.fill_(-7)
            assert all(torch.equal(u, v) for j, (u, v) in enumerate(zip(first, before)) if j != i)
            assert torch.equal(torch.clone(want), before[i])
        kept = first[1]
        del first
        assert bool((kept == -7).all())
    cache, users, table, lengths, _ = made["fork"][1]
    empty = F.cache_fork(cache, users, table[:0], lengths[:0], lengths[:0])
    assert torch.equal(empty[0], users) and empty[1].shape == (0, 3) and empty[2].shape == (0,)


def test_closed_and_new_contexts(calls):
    """A closed context is refused by every call, and one in its place takes them over, with what is told of them."""
    import torch
    import frisk_b200 as F
    made = arguments()
    want = {name: flat(made[name][0](*made[name][1])) for name in ("verify", "adapters", "fork", "grow", "compact", "keep")}
    F.cache_check()
    held = calls.execute._contexts
    mine = held[0]
    address = calls.address(0)
    mine.close()
    try:
        assert address and calls.address(0) is None
        for function, args, native, native_args in made.values():
            assert native(*native_args) is None
            with pytest.raises(RuntimeError, match="destroyed"):
                function(*args)
    finally:
        del held[0]
    again = arguments()
    for name, results in want.items():
        assert all(torch.equal(a, b) for a, b in zip(flat(again[name][0](*again[name][1])), results)), name
    assert calls.address(0) == held[0].handle.value
    F.cache_check()
    _, args, native, native_args = again["keep"]
    assert native(*native_args[:-1], ints([99, 99])) is not None
    with pytest.raises(RuntimeError, match="table"):
        F.cache_check()


def test_what_results_keep(calls):
    """Of a verification each its own memory; of new tables no more than the three and the scratch that the documentation names."""
    made = arguments()
    function, args, _, _ = made["verify"]
    kept, counts, token = function(*args)
    storages = [t.untyped_storage() for t in (kept, counts, token)]
    assert len({s.data_ptr() for s in storages}) == 3
    assert [s.nbytes() for s in storages] == [t.numel() * t.element_size() for t in (kept, counts, token)]
    for name in ("fork", "grow", "compact"):
        function, args, _, _ = made[name]
        results = function(*args)
        total = sum(-(-t.numel() * 4 // 64) * 64 for t in results)
        assert all(t.untyped_storage().nbytes() <= total + (1 << 16) for t in results)
        assert results[2].clone().untyped_storage().nbytes() == results[2].numel() * 4
