"""The serving operators together, as a server runs them: prompts, samples that fork, drafted trees that are scored, verified and settled, beams that
change places, a cache that is compacted, copied and shrunk; each request with its own adapter.  What the cache holds is compared with
what was written, key by key, after every step."""
import random

import pytest

from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu


class Server:
    HEADS, GROUP, D, MODEL, VOCAB, RANK = 2, 2, 64, 128, 211, 8

    def __init__(self, held, batch, pages, width, page, seed):
        import torch
        import frisk_b200 as F
        self.F, self.torch, self.page, self.rng = F, torch, page, random.Random(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g = g
        self.cache = F.paged_cache(pages, self.HEADS, page, self.D, getattr(torch, held))
        self.users, self.table, self.lengths = F.page_tables(self.cache, batch, width)
        h = (self.HEADS * self.GROUP + 2 * self.HEADS) * self.D
        mk = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).bfloat16()  # noqa: E731
        self.w, self.a, self.b = mk(h, self.MODEL, scale=self.MODEL ** -0.5), mk(3, self.RANK, self.MODEL, scale=0.1), mk(3, h, self.RANK, scale=0.5)
        self.frequencies, _ = F.rotary_frequencies(self.D)
        self.which = torch.tensor([self.rng.randint(-1, 2) for _ in range(batch)], dtype=torch.int32, device="cuda")
        self.history = [[] for _ in range(batch)]  # of every sequence: the (key, value) rows it should hold, on the host
        self.batch = batch

    def rows(self, counts, positions):
        """Queries, keys and values of new tokens, and starts."""
        F, torch = self.F, self.torch
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        x = (torch.randn(starts[-1], self.MODEL, generator=self.g, device="cuda")).bfloat16()
        starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        y = torch.empty(len(x), len(self.w), dtype=torch.bfloat16, device="cuda")
        F.gemm(x, self.w, y, trans_b=True)
        plain = y.clone()
        y = F.adapter_gemm(x, self.a, self.b, y, starts, self.which)
        want, bound = so.adapters(x.cpu(), self.a.cpu(), self.b.cpu(), plain.cpu(), starts.tolist(), self.which.tolist())
        assert float(((y.cpu().double() - want).abs() - bound).max()) <= 0
        hq, hk = self.HEADS * self.GROUP, self.HEADS
        q, k, v = (t.view(len(x), -1, self.D) for t in y.split([hq * self.D, hk * self.D, hk * self.D], 1))
        q, k = F.rotary(q, k, torch.tensor(positions, device="cuda"), self.frequencies)
        return q, k, v, starts

    def check(self):
        """The tables are what they should be, and the cache holds what was written."""
        F, torch = self.F, self.torch
        F.cache_check()
        lengths, table, users = self.lengths.tolist(), self.table.tolist(), self.users.tolist()
        assert lengths == [len(h) for h in self.history]
        count = [0] * len(users)
        for row in table:
            for p in row:
                if p >= 0:
                    count[p] += 1
        assert count == users
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        if starts[-1] == 0:
            return
        k, v = F.cache_read(self.cache, self.table, torch.tensor(starts, dtype=torch.int32, device="cuda"), torch.zeros_like(self.lengths), starts[-1], dtype=torch.bfloat16)
        want = [row for h in self.history for row in h]
        assert torch.equal(k.cpu(), torch.stack([r[0] for r in want])) and torch.equal(v.cpu(), torch.stack([r[1] for r in want]))

    def held(self, k, v):
        """Rows as the cache gives them back."""
        F, torch = self.F, self.torch
        n = len(k)
        if self.cache[0].dtype == torch.bfloat16:
            return list(zip(k.cpu(), v.cpu()))
        spare = F.paged_cache(-(-n // 16), self.HEADS, 16, self.D, self.cache[0].dtype)
        table, starts, none = torch.arange(-(-n // 16), dtype=torch.int32, device="cuda")[None], torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        F.cache_write(spare, k, v, table, starts, none)
        return list(zip(*(t.cpu() for t in F.cache_read(spare, table, starts, none, n, dtype=torch.bfloat16))))

    def grow(self, starts):
        self.users, self.table, granted = self.F.cache_grow(self.cache, self.users, self.table, starts, self.lengths)
        counts = [b - a for a, b in zip(starts.tolist(), starts.tolist()[1:])]
        assert granted.tolist() == counts
        return counts

    def prompts(self, counts):
        positions = [len(h) + i for h, n in zip(self.history, counts) for i in range(n)]
        q, k, v, starts = self.rows(counts, positions)
        self.grow(starts)
        self.F.cache_write(self.cache, k, v, self.table, starts, self.lengths)
        self.F.cache_attention(self.cache, q, self.table, starts, self.lengths)
        rows = self.held(k, v)
        for b, (first, n) in enumerate(zip(starts.tolist(), counts)):
            self.history[b] += rows[first:first + n]
        self.lengths = self.lengths + torch_counts(counts)
        self.check()

    def fork(self, parents):
        self.users, self.table, self.lengths = self.F.cache_fork(self.cache, self.users, self.table, self.lengths, torch_counts(parents))
        self.history = [list(self.history[p]) if p >= 0 else [] for p in parents]
        self.check()

    def step(self, most):
        """Trees of drafted tokens behind the last one: scored, verified, settled."""
        F, torch = self.F, self.torch
        counts = [self.rng.randint(1, most) if h else 0 for h in self.history]
        parents, depth, starts = [], [], [0]
        for n in counts:
            mine = [-1] + [self.rng.randrange(i) for i in range(1, n)]
            deep = []
            for p in mine[:n]:
                deep.append(0 if p < 0 else deep[p] + 1)
            parents += mine[:n]
            depth += deep
            starts.append(starts[-1] + n)
        owner = [b for b, n in enumerate(counts) for _ in range(n)]
        q, k, v, starts_gpu = self.rows(counts, [len(self.history[b]) + d for b, d in zip(owner, depth)])
        mask = torch.zeros(len(owner), most, dtype=torch.bool)
        for r, b in enumerate(owner):
            i = r - starts[b]
            if parents[r] >= 0:
                mask[r] = mask[starts[b] + parents[r]]
            mask[r, i] = True
        self.grow(starts_gpu)
        F.cache_write(self.cache, k, v, self.table, starts_gpu, self.lengths)
        out = F.cache_attention(self.cache, q, self.table, starts_gpu, self.lengths, mask=mask.cuda(), max_new=most)
        assert bool(torch.isfinite(out).all())
        logits = torch.randn(len(owner), self.VOCAB, generator=self.g, device="cuda") * 3
        target, draft = torch.softmax(logits, -1), torch.softmax(logits + torch.randn(logits.shape, generator=self.g, device="cuda"), -1)
        tokens = torch.multinomial(draft[[starts[b] + max(0, parents[r]) for r, b in enumerate(owner)]], 1, generator=self.g)[:, 0]
        accept, sample = torch.rand(len(owner), generator=self.g, device="cuda"), torch.rand(self.batch, generator=self.g, device="cuda")
        p = torch_counts(parents)
        kept, many, token = F.draft_verify(tokens, p, starts_gpu, target, draft, accept, sample, max_new=most)
        want = so.verify(tokens.tolist(), parents, starts, target.cpu(), draft.cpu(), accept.tolist(), sample.tolist(), most)
        assert [kept.tolist(), many.tolist(), token.tolist()] == list(want)
        self.lengths = F.cache_keep(self.cache, self.table, starts_gpu, self.lengths, kept, many)
        rows = self.held(k, v)
        for b, n in enumerate(want[1]):
            self.history[b] += [rows[starts[b] + i] for i in want[0][b][:n]]
        self.check()

    def compact(self):
        self.users, self.table, used = self.F.cache_compact(self.cache, self.users, self.table)
        n = int(used)
        assert bool((self.users[:n] > 0).all()) and not bool(self.users[n:].any())
        self.check()
        return n

    def move(self, pages):
        """Into a cache of another size."""
        F, torch = self.F, self.torch
        n = self.compact()
        new = F.paged_cache(pages, self.HEADS, self.page, self.D, self.cache[0].dtype)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:n].int().cuda()
        F.cache_copy(self.cache, torch.arange(n, dtype=torch.int32, device="cuda"), order, into=new)
        users = torch.zeros(pages, dtype=torch.int32, device="cuda")
        users[order.long()] = self.users[:n]
        self.table = torch.where(self.table < 0, self.table, order[self.table.clamp(min=0).long()])
        self.cache, self.users = new, users
        self.check()


def torch_counts(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("held", ["bfloat16", "float8_e4m3fn"])
@pytest.mark.parametrize("page", [16, 64])
def test_a_server(held, page):
    s = Server(held, 6, 80, 20, page, 3)
    s.prompts([37, 0, 90, 0, 5, 0])
    s.fork([0, 0, 2, 2, 4, 0])       # samples of two prompts
    s.step(6)
    s.step(9)
    s.fork([1, 0, 3, 3, -1, 5])      # beams change places, one request ends
    s.step(5)
    s.prompts([0, 0, 0, 0, 70, 1])   # another takes its place
    s.compact()
    s.step(7)
    s.move(60)
    s.step(4)
    s.fork(list(range(6)))           # pages behind the last key come back
    s.step(1)
    s.fork([-1] * 6)
    assert not bool(s.users.any())
