"""Verification of drafted tokens against oracle/serving_oracle.py: the same nodes and the same token."""
import math

import pytest

from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu


class Drafts:
    """Trees (or chains) of drafted tokens over random distributions; the draft's are near the target's."""

    def __init__(self, counts, vocab, dtype="float32", draft=True, tree=True, seed=0, gap=0, pitch=0, sharp=2.0):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.starts = [gap]
        for n in counts:
            self.starts.append(self.starts[-1] + n)
        rows = self.starts[-1] + gap
        logits = torch.randn(rows, vocab, generator=g) * sharp

        def held(x):
            whole = torch.full((rows, vocab + pitch), math.nan, dtype=getattr(torch, dtype))
            whole[:, :vocab] = torch.softmax(x, -1).to(whole.dtype)
            return whole[:, :vocab]

        self.target = held(logits)
        self.draft = held(logits + 0.7 * torch.randn(rows, vocab, generator=g)) if draft else None
        self.tree = tree
        self.parents = [0] * rows
        tokens = torch.zeros(rows, dtype=torch.int64)
        source = self.target if self.draft is None else self.draft
        for first, n in zip(self.starts, counts):
            for i in range(n):
                up = -1 if i == 0 else max(0, i - int(torch.randint(1, 6, (1,), generator=g))) if tree else i - 1
                self.parents[first + i] = up
                if i:
                    tokens[first + i] = torch.multinomial(source[first + up].float().clone(), 1, generator=g)[0]
        self.tokens = tokens
        self.accept, self.sample = torch.rand(rows, generator=g), torch.rand(len(counts), generator=g)
        self.max_new = max(counts + [1])

    def run(self, max_new=None, tokens=None, stream=None):
        import torch
        import frisk_b200 as F

        def place(t):  # the pitch stays
            return None if t is None else t if t.is_cuda else t._base.cuda()[:, :t.shape[1]] if t._base is not None and t.dim() == 2 else t.cuda()

        tokens = self.tokens if tokens is None else tokens
        parents = torch.tensor(self.parents, dtype=torch.int32).cuda() if self.tree else None
        got = F.draft_verify(tokens.cuda(), parents, torch.tensor(self.starts, dtype=torch.int32).cuda(), place(self.target), place(self.draft), self.accept.cuda(),
                             self.sample.cuda(), max_new=max_new or self.max_new, stream=stream)
        assert got[2].dtype == tokens.dtype
        return [t.tolist() for t in got]

    def want(self, max_new=None):
        return list(so.verify(self.tokens.tolist(), self.parents if self.tree else None, self.starts, self.target, self.draft, self.accept.tolist(), self.sample.tolist(),
                              max_new or self.max_new))


@pytest.mark.parametrize("counts,vocab", [([1], 1), ([1, 1], 3), ([4], 2), ([5, 0, 9, 1], 7), ([6] * 9, 256), ([3, 8], 257), ([2, 5], 2047), ([24, 17], 5001), ([40], 33000), ([7], 131072)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("tree", [False, True])
def test_verify(counts, vocab, dtype, draft, tree):
    import frisk_b200 as F
    d = Drafts(counts, vocab, dtype, draft, tree, seed=vocab, pitch=vocab % 3, gap=vocab % 2)
    assert d.run() == d.want()
    assert d.run(max_new=d.max_new + 3) == d.want(d.max_new + 3)
    F.cache_check()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [100, 4099])
def test_the_draft_in_rows_of_another_pitch(dtype, vocab):
    """Rows of the two begin at other places of 16 bytes."""
    import torch
    d = Drafts([9, 6, 12], vocab, dtype, seed=7, pitch=1)
    for more in (0, 2, 5):
        whole = torch.full((len(d.draft), vocab + more), math.nan, dtype=d.draft.dtype)
        whole[:, more // 2:more // 2 + vocab] = d.draft
        target, d.draft = d.draft, whole[:, more // 2:more // 2 + vocab]
        import frisk_b200 as F
        wide = whole.cuda()
        got = F.draft_verify(d.tokens.cuda(), torch.tensor(d.parents, dtype=torch.int32).cuda(), torch.tensor(d.starts, dtype=torch.int32).cuda(),
                             d.target._base.cuda()[:, :vocab], wide[:, more // 2:more // 2 + vocab], d.accept.cuda(), d.sample.cuda(), max_new=12)
        assert [t.tolist() for t in got] == d.want()
        d.draft = target
    F.cache_check()


def test_many_seeds_and_types_of_tokens():
    """Every kind of walk: all stand, none does, several children of a node fall, the same child twice."""
    import torch
    seen = set()
    for seed in range(30):
        d = Drafts([1 + (seed * 5 + i) % 9 for i in range(12)], 5 + seed % 3, draft=seed % 2 == 0, seed=seed, sharp=1.0)
        got = d.run()
        assert got == d.want(), seed
        seen |= set(got[1])
        d.tokens = d.tokens.int()
        assert d.run() == got
    assert seen >= {1, 2, 3, 4}


def test_borders():
    """Exact ties: u at a border takes the token behind it; u below 1 never runs past the last token that weighs anything."""
    import torch
    d = Drafts([1, 1, 1, 1, 1], 8, draft=False)
    d.target[:] = torch.tensor([0.0, 0.25, 0.0, 0.25, 0.5, 0.0, 0.0, 0.0])
    d.sample = torch.tensor([0.0, 0.25, 0.49999997, 0.5, 0.99999994])
    got = d.run()
    assert got[2] == [1, 3, 3, 4, 4] and got == d.want()
    # acceptance is strict: u q < w
    d = Drafts([2, 2, 2, 2], 4, tree=False)
    d.target[:] = torch.tensor([0.25, 0.5, 0.25, 0.0])
    d.draft[:] = torch.tensor([0.5, 0.25, 0.0, 0.25])
    d.tokens[:] = torch.tensor([0, 0, 0, 0, 0, 2, 0, 3])
    d.accept = torch.tensor([0, 0.5, 0, 0.49999997, 0, 0.99999994, 0, 0.0])  # at the ratio; below it; not the draft's at all; impossible
    d.sample = torch.tensor([0.49999997, 0.0, 0.0, 0.5])
    got = d.run()
    assert got[1] == [1, 2, 2, 1] and got == d.want()


def test_odd_probabilities():
    """NaN and negative values weigh nothing, infinities the largest finite value; rows that are empty, or end up empty."""
    import torch
    for draft in (False, True):
        d = Drafts([3, 3, 3, 3, 2], 700, draft=draft, tree=False, seed=9)
        d.target[0, 10:600] = math.nan
        d.target[1] = -1.0
        d.target[3] = 0.0
        d.target[4] = math.nan
        d.target[6, 5] = math.inf
        d.target[9:12] = 0.0
        d.target[9:12, 699] = 2.0
        if draft:
            d.draft[0, 100:300] = math.nan
            d.draft[9:12] = d.target[9:12]   # nothing is left of it
            d.draft[12] = math.inf
        d.tokens[10:12] = 699
        d.accept[10] = 0.999
        got = d.run()
        assert got == d.want()
        assert got[2][1] == -1 and got[2][2] == 5 or got[1][2] > 1
    # every row empty: no token
    d = Drafts([2, 1], 300, draft=False)
    d.target[:] = 0
    assert d.run() == [[[0, -1], [0, -1]], [1, 1], [-1, -1]]


def test_trees_as_they_come():
    """Parents that are no node before their child, tokens outside the vocabulary: they do not stand, nor does what follows them."""
    import torch
    d = Drafts([6, 6], 50, draft=False, seed=2)
    d.parents = [-1, 0, 0, 9, 3, -5, 0, 0, 2, 1, 3, 3]
    d.tokens[1] = 50
    d.tokens[7] = -1
    d.accept[:] = 0
    assert d.run() == d.want()
    d.tokens[2] = 1 << 40
    assert d.run() == d.want()


def test_offsets_beyond_32_bits():
    """Rows behind the first 2^31 values: as those rows by themselves."""
    import torch
    import frisk_b200 as F
    rows, vocab, n = 12000, 200000, 9
    both = [torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    torch.manual_seed(3)
    for t in both:
        t[-n:] = torch.rand(n, vocab, device="cuda").bfloat16()
    tokens, accept, sample = torch.randint(0, vocab, (rows,), device="cuda"), torch.rand(rows, device="cuda"), torch.rand(2, device="cuda")
    starts = torch.tensor([rows - n, rows - 4, rows], dtype=torch.int32, device="cuda")
    for draft in (False, True):
        got = F.draft_verify(tokens, None, starts, both[0], both[1] if draft else None, accept, sample, max_new=6)
        few = F.draft_verify(tokens[-n:].clone(), None, starts - (rows - n), both[0][-n:].clone(), both[1][-n:].clone() if draft else None, accept[-n:].clone(), sample, max_new=6)
        F.cache_check()
        assert all(torch.equal(a, b) for a, b in zip(got, few)) and bool((got[2] >= 0).all())


def test_rows_out_of_range_are_left_out():
    import frisk_b200 as F
    d = Drafts([3, 5, 2], 40)
    got, want = d.run(max_new=4), d.want(4)
    with pytest.raises(RuntimeError, match="table"):
        F.cache_check()
    assert got == want and got[1][1] == 0 and got[2][1] == -1
    right = d.run()
    for starts in ([-1, 3, 8, 10], [0, 8, 3, 10], [0, 3, 8, 11], [0, 3, 8, -(1 << 31)]):
        d.starts = starts
        got = d.run()
        with pytest.raises(RuntimeError, match="table"):
            F.cache_check()
        fine = [0 <= a <= b <= 10 and b - a <= d.max_new for a, b in zip(starts, starts[1:])]
        assert [n > 0 for n in got[1]] == [f and b > a for f, a, b in zip(fine, starts, starts[1:])]
        for b in range(3):
            if fine[b] and starts[b:b + 2] == [0, 3, 8, 10][b:b + 2]:
                assert [x[b] for x in got] == [x[b] for x in right]
    F.cache_check()


def test_the_targets_distribution_comes_out():
    """Children drawn from the draft, whatever it is: the first token behind the root has the target's distribution, to six deviations."""
    import torch
    import frisk_b200 as F
    g = torch.Generator(device="cuda").manual_seed(11)
    n, vocab = 16000, 6
    p = torch.tensor([0.4, 0.05, 0.25, 0.0, 0.2, 0.1], device="cuda")
    q = torch.tensor([0.1, 0.5, 0.1, 0.1, 0.1, 0.1], device="cuda")
    for draft, children in ((q, 3), (None, 2)):
        rows = n * (children + 1)
        tokens = torch.multinomial(p if draft is None else draft, rows, replacement=True, generator=g)
        if draft is None:  # picked, not drawn: always the same two
            tokens = torch.tensor([0, 1, 2], device="cuda").repeat(n)
        parents = torch.tensor([-1] + [0] * children, dtype=torch.int32, device="cuda").repeat(n)
        starts = torch.arange(n + 1, dtype=torch.int32, device="cuda") * (children + 1)
        kept, counts, token = F.draft_verify(tokens, parents, starts, p.expand(rows, vocab), None if draft is None else draft.expand(rows, vocab),
                                             torch.rand(rows, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda"), max_new=children + 1)
        first = torch.where(counts > 1, tokens.view(n, -1).gather(1, kept[:, 1:2].long().clamp(min=0))[:, 0], token)
        for have, want in zip((torch.bincount(first, minlength=vocab) / n).tolist(), p.tolist()):
            assert abs(have - want) <= 6 * (want * (1 - want) / n) ** 0.5
    F.cache_check()


def test_refusals_streams_and_graphs():
    import torch
    import frisk_b200 as F
    d = Drafts([3, 4], 1000)
    args = [d.tokens.cuda(), torch.tensor(d.parents, dtype=torch.int32).cuda(), torch.tensor(d.starts, dtype=torch.int32).cuda(), d.target.cuda(), d.draft.cuda(), d.accept.cuda(),
            d.sample.cuda()]

    def call(i=None, x=None, max_new=4, **more):
        return F.draft_verify(*[x if j == i else a for j, a in enumerate(args)], max_new=max_new, **more)

    for bad in ((0, args[0].float()), (0, args[0][:6]), (0, args[0].cpu()), (1, args[1].long()), (1, args[1][:3]), (2, args[2].long()), (2, args[2][None]), (3, args[3].double()),
                (3, args[3][0]), (3, args[3].t().contiguous().t()), (4, args[4].half()), (4, args[4][:, :9]), (5, args[5].double()), (5, args[5][:2]), (6, args[6][:1]),
                (6, args[6].half())):
        with pytest.raises(ValueError):
            call(*bad)
    for n in (0, -1, 1025):
        with pytest.raises(ValueError):
            call(max_new=n)
    want = d.want()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = call(stream=side)
    side.synchronize()
    assert [t.tolist() for t in got] == want
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (5, 6):
        other = Drafts([3, 4], 1000, seed=seed)
        for a, b in zip(args, [other.tokens, torch.tensor(other.parents, dtype=torch.int32), torch.tensor(other.starts, dtype=torch.int32), other.target, other.draft, other.accept,
                               other.sample]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert [t.tolist() for t in got] == other.want()
    # no sequences, or none with rows
    none = F.draft_verify(args[0][:0], None, args[2][:1] * 0, args[3][:0], None, args[5][:0], args[6][:0], max_new=3)
    assert [list(t.shape) for t in none] == [[0, 3], [0], [0]]
    got = F.draft_verify(args[0][:0], None, args[2] * 0, args[3][:0], None, args[5][:0], args[6], max_new=3)
    assert [t.tolist() for t in got] == [[[-1] * 3] * 2, [0, 0], [-1, -1]]
    F.cache_check()
