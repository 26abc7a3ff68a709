"""Performance cases of what a server does around its projections and its paged cache.

Three groups of operators: ``draft_verify``; the pages of a cache (``cache_fork``, ``cache_grow``, ``cache_keep``, ``cache_copy``,
``cache_compact``); ``adapter_gemm``.  A case names its kind:

* ``verify``    which drafted tokens stand, and the token after them, from given random numbers
* ``settle``    the same behind a write of the drafted rows, then the accepted rows moved together in the cache
* ``branch``    sequences that share pages (samples of a prompt, beams that are reordered, some that end), then room for the next tokens
* ``copy``      pages copied into another cache
* ``compact``   used pages moved to the lowest indices
* ``adapters``  the low-rank adapters of many requests added to a shared projection

Packed rows: sequence b's new tokens are rows starts[b] .. starts[b + 1] - 1, and lengths[b] keys of it are in the cache before them.
A cache is (k, v) of [pages, heads, page, D], with an 8-bit exponent for every token and head where it holds 8-bit floats.
"""
import math
import random

import torch

own = False

_DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
_SIZE = {"fp16": 2, "bf16": 2, "fp32": 4, "e4m3": 1}


def _verify(b, new, vocab, dtype, draft, tree, kind="verify", **name):
    """``new``: nodes of a sequence at most, the last sampled token among them; ``draft``: the draft's distributions are given."""
    return dict(name, kind=kind, b=b, new=new, vocab=vocab, dtype=dtype, draft=draft, tree=tree)


def _settle(b, new, vocab, draft, tree, length, hkv, d, page, rows, held, **name):
    return dict(_verify(b, new, vocab, "fp32", draft, tree, "settle", **name), length=length, hkv=hkv, d=d, page=page, rows=rows, held=held)


def _branch(groups, each, ended, length, new, hkv, d, page, held, **name):
    """``groups`` requests of ``each`` sequences; ``ended`` of the requests end; lengths up to ``length``, ``new`` tokens each at most."""
    return dict(name, kind="branch", groups=groups, each=each, ended=ended, length=length, new=new, hkv=hkv, d=d, page=page, held=held)


def _pages(kind, pages, moved, hkv, d, page, held, **name):
    """``moved``: pages that are copied, or that are in use, of ``pages``."""
    return dict(name, kind=kind, pages=pages, moved=moved, hkv=hkv, d=d, page=page, held=held)


def _adapters(b, new, count, rank, k, n, dtype, out, **name):
    """``b`` requests of up to ``new`` tokens over ``count`` adapters; ``out``: type of the projection's result."""
    return dict(name, kind="adapters", b=b, new=new, count=count, rank=rank, k=k, n=n, dtype=dtype, out=out)


def listed():
    return [
        # one sequence, four tokens guessed from its own past: all latency
        _verify(1, 5, 32000, "fp32", False, False, name="verify_one_chain"),
        # a batch with a draft model, five tokens each
        _verify(64, 6, 128000, "fp32", True, False, name="verify_chains"),
        # trees of 24 nodes, several children a node, 16-bit probabilities over an odd vocabulary
        _verify(16, 24, 50001, "bf16", True, True, name="verify_trees_odd"),
        # behind the attention of a step: trees written, verified, and the accepted path moved together in an 8-bit cache
        _settle(24, 25, 32000, False, True, 2000, 8, 128, 16, "bf16", "e4m3", name="settle_trees_e4m3"),
        # sixteen samples of one prompt: pages shared, the last one copied for each
        _branch(1, 16, 0, 2000, 1, 8, 128, 64, "bf16", name="branch_samples"),
        # beams of 48 requests change places, some requests end, and all go on by up to five tokens
        _branch(48, 4, 3, 6000, 5, 8, 128, 16, "e4m3", name="branch_beams_e4m3"),
        # the sequences of preempted requests brought into another cache
        _pages("copy", 1600, 1400, 8, 128, 64, "bf16", name="copy_bf16"),
        # a cache that emptied to a third, before it is made smaller
        _pages("compact", 9000, 3001, 4, 64, 64, "e4m3", name="compact_e4m3"),
        # one token of one request: all latency
        _adapters(1, 1, 4, 16, 4096, 4096, "bf16", "bf16", name="adapters_one_token"),
        # a batch that decodes, 64 requests over 40 adapters
        _adapters(64, 1, 40, 32, 4096, 5120, "bf16", "bf16", name="adapters_decode"),
        # drafted tokens, odd widths, products left in 32 bits
        _adapters(24, 5, 24, 8, 5000, 2500, "fp16", "fp32", name="adapters_drafts_odd"),
        # prompts of eight requests
        _adapters(8, 1024, 6, 64, 4096, 8192, "bf16", "bf16", name="adapters_prompts"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "settle", "branch", "branch", "copy", "compact", "adapters", "adapters", "adapters"])
    if kind == "adapters":
        new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 2048)])
        b = _log(rng, 1, max(1, min(128, 8192 // new)))
        k, n = (rng.choice([1024, 2048, 4096, 8192, 8 * rng.randint(16, 1024), 4 * rng.randint(32, 2000)]) for _ in (0, 1))
        dtype = rng.choice(["bf16", "fp16"])
        return _adapters(b, new, _log(rng, 1, 48), rng.choice([8, 16, 16, 24, 32, 64, 128]), k, n if b * new < 4096 else min(n, 8192), dtype,
                         rng.choice([dtype, dtype, "fp32"]))
    if kind == "verify":
        vocab = _log(rng, 1000, 160000)
        b = _log(rng, 1, 64)
        new = _log(rng, 1, max(2, min(64, 48000000 // (b * vocab))))
        return _verify(b, new, vocab, rng.choice(["fp32", "fp32", "bf16", "fp16"]), rng.random() < 0.6, rng.random() < 0.5)
    hkv, d, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if kind == "settle":
        b, rows = _log(rng, 1, 64), rng.choice(["bf16", "fp16"])
        return _settle(b, _log(rng, 1, 32), rng.choice([8000, 32000]), rng.random() < 0.3, rng.random() < 0.6, _log(rng, 1, 2000), hkv, d, page, rows,
                       rng.choice([rows, "e4m3"]))
    held = rng.choice(["bf16", "fp16", "e4m3"])
    if kind == "branch":
        groups = _log(rng, 1, 64)
        return _branch(groups, _log(rng, 1, 16) if groups < 16 else rng.randint(1, 4), rng.randint(0, groups // 4), _log(rng, 1, 200000 // groups if groups > 30 else 6000),
                       _log(rng, 1, 64), hkv, d, page, held)
    size = hkv * d * page * 2 * _SIZE[held]  # of a page, keys and values
    pages = _log(rng, 2, min(40000, 600000000 // size))
    return _pages(kind, pages, rng.randint(1, max(1, pages * 7 // 8)), hkv, d, page, held)


# ---------------------------------------------------------------------------------------- inputs
def _ragged(c):
    """Tokens and keys of every sequence: between two thirds and all of the largest count, by the case alone."""
    rng = random.Random(c["b"] * 1000003 + c["new"] * 1009 + c.get("length", 0))
    if c["b"] == 1:
        return [c["new"]], [c.get("length", 0)]
    counts = [rng.randint(max(1, 2 * c["new"] // 3), c["new"]) for _ in range(c["b"])]
    return counts, [rng.randint(2 * c.get("length", 0) // 3, c.get("length", 0)) for _ in range(c["b"])]


def _starts(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


def _ints(x, dev="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _new_cache(pages, c, g, dev="cuda"):
    shape = (pages, c["hkv"], c["page"], c["d"])
    if c["held"] != "e4m3":
        return tuple(torch.randn(shape, generator=g, device=dev, dtype=_DTYPE[c["held"]]) for _ in (0, 1))

    def codes():
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float16).mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)

    return (codes(), codes()) + tuple(torch.randint(117, 121, shape[:3], generator=g, device=dev, dtype=torch.uint8) for _ in (0, 1))


def _prepare_drafts(c, gen, g, dev):
    counts, lengths = _ragged(c)
    starts, dt = _starts(counts), _DTYPE[c["dtype"]]
    total = starts[-1]
    parents = []
    for n in counts:
        back = torch.randint(1, 9, (n,), generator=gen).tolist()
        parents += [-1 if i == 0 else max(0, i - back[i]) if c["tree"] else i - 1 for i in range(n)]
    at = torch.tensor([starts[b] + max(0, parents[starts[b] + i]) for b, n in enumerate(counts) for i in range(n)], device=dev)  # row of a node's parent
    # the target's distributions, and a draft's that are near them; drafted tokens come from the draft's, or are mostly likely ones
    logits = torch.randn(total, c["vocab"], generator=g, device=dev).mul_(3.0)
    target = torch.softmax(logits, -1).to(dt)
    draft = torch.softmax(logits.add_(torch.randn(logits.shape, generator=g, device=dev).mul_(0.6)), -1).to(dt) if c["draft"] else None
    if draft is None:
        target = torch.softmax(logits.mul_(2.0), -1).to(dt)
    tokens = torch.empty(total, dtype=torch.int64, device=dev)
    for first in range(0, total, 64):
        rows = at[first:first + 64]
        tokens[first:first + 64] = torch.multinomial((target if draft is None else draft)[rows].float(), 1, generator=g)[:, 0]
    return dict(c, counts=counts, lengths_host=lengths, starts_host=starts, total=total, target=target, draft=draft, tokens=tokens,
                parents=_ints(parents), starts=_ints(starts), accept=torch.rand(total, generator=g, device=dev),
                sample=torch.rand(c["b"], generator=g, device=dev))


def _group_lengths(c):
    """Of every request's sequences: keys (the beams of a request are as long as one another), and new tokens."""
    rng = random.Random(c["groups"] * 7919 + c["length"] * 31 + c["new"])
    lengths = [c["length"] if c["groups"] == 1 else rng.randint(max(1, 2 * c["length"] // 3), c["length"]) for _ in range(c["groups"])]
    return lengths, [rng.randint(max(1, 2 * c["new"] // 3), c["new"]) for _ in range(c["groups"])]


def _branch_plan(c):
    """(parents, new tokens of every sequence) by the case alone: a request's beams take one another's places, a request that ends gives
    its pages back, and samples of a single prompt all come from the first."""
    rng = random.Random(c["groups"] * 104729 + c["each"] * 271 + c["new"])
    _, new = _group_lengths(c)
    gone = set(rng.sample(range(c["groups"]), min(c["ended"], c["groups"] - 1)))
    parents, counts = [], []
    for g in range(c["groups"]):
        for _ in range(c["each"]):
            parents.append(-1 if g in gone else g * c["each"] + (0 if c["groups"] == 1 else rng.randrange(c["each"])))
            counts.append(0 if g in gone else new[g])
    return parents, counts


def _prepare_branch(c, gen, g, dev):
    page, each = c["page"], c["each"]
    lengths, new = _group_lengths(c)
    parents, counts = _branch_plan(c)
    b = c["groups"] * each
    need = [-(-n // page) for n in lengths]
    width = max(-(-(n + m) // page) for n, m in zip(lengths, new)) + 2
    # the beams of a request share all but their last two pages, of which every beam has its own
    single = c["groups"] == 1
    held = sum(need) if single else sum(max(0, n - 2) + each * min(n, 2) for n in need)
    pages = held + sum(-(-m // page) + 2 for m in new) * each + 8
    order = torch.randperm(pages, generator=gen).tolist()
    users, table, lens = [0] * pages, [[-1] * width for _ in range(b)], [0] * b
    at = 0
    for i, n in enumerate(need):
        if single:
            rows, shared = [0], 0
        else:
            rows, shared = range(i * each, (i + 1) * each), max(0, n - 2)
        common = order[at:at + shared]
        at += shared
        for r in rows:
            mine = order[at:at + n - shared]
            at += n - shared
            table[r][:n] = common + mine
            lens[r] = lengths[i]
            for p in common + mine:
                users[p] += 1
    return dict(c, cache=_new_cache(pages, c, g), users=_ints(users), table=_ints(table), lengths=_ints(lens), parents=_ints(parents),
                starts=_ints(_starts(counts)), width=width)


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    c = dict(case)
    if c["kind"] == "verify":
        return _prepare_drafts(c, gen, g, dev)
    if c["kind"] == "settle":
        s = _prepare_drafts(c, gen, g, dev)
        need = [-(-(n + m) // c["page"]) for n, m in zip(s["lengths_host"], s["counts"])]
        pages = sum(need) + 8
        order = torch.randperm(pages, generator=gen).tolist()
        table = [[-1] * max(need) for _ in need]
        for b, n in enumerate(need):
            table[b][:n] = [order.pop() for _ in range(n)]
        rows = torch.randn(s["total"], 2 * c["hkv"] * c["d"], generator=g, device=dev).to(_DTYPE[c["rows"]])
        k, v = (rows[:, i * c["hkv"] * c["d"]:(i + 1) * c["hkv"] * c["d"]].view(-1, c["hkv"], c["d"]) for i in (0, 1))
        return dict(s, cache=_new_cache(pages, c, g), table=_ints(table), lengths=_ints(s["lengths_host"]), k=k, v=v)
    if c["kind"] == "branch":
        return _prepare_branch(c, gen, g, dev)
    if c["kind"] == "copy":
        # into a cache of another size, in another order
        other = c["moved"] + c["pages"] // 8
        return dict(c, cache=_new_cache(c["pages"], c, g), into=_new_cache(other, c, g), source=torch.randperm(c["pages"], generator=gen)[:c["moved"]].int().to(dev),
                    target=torch.randperm(other, generator=gen)[:c["moved"]].int().to(dev))
    if c["kind"] == "compact":
        order = torch.randperm(c["pages"], generator=gen)[:c["moved"]].int()
        width = min(128, c["moved"])
        table = torch.full((-(-c["moved"] // width), width), -1, dtype=torch.int32)
        table.view(-1)[:c["moved"]] = order
        users = torch.zeros(c["pages"], dtype=torch.int32)
        users[order.long()] = 1
        return dict(c, cache=_new_cache(c["pages"], c, g), users=users.to(dev), table=table.to(dev))
    counts, _ = _ragged(c)
    starts, dt = _starts(counts), _DTYPE[c["dtype"]]

    def padded(n, cols, scale, to):  # rows on 16 bytes, as an allocator of weights lays them out
        return torch.randn(n, -(-cols // 8) * 8, generator=g, device=dev).mul_(scale).to(to)[:, :cols]

    a = padded(c["count"] * c["rank"], c["k"], c["k"] ** -0.5, dt).unflatten(0, (c["count"], c["rank"]))
    b = torch.randn(c["count"], c["n"], c["rank"], generator=g, device=dev).mul_(0.5).to(dt)
    which = torch.randint(0, c["count"], (c["b"],), generator=gen, dtype=torch.int32)
    if c["b"] > 8:  # some requests have none
        which[torch.randperm(c["b"], generator=gen)[:c["b"] // 12]] = -1
    return dict(c, x=padded(starts[-1], c["k"], 1.0, dt), a=a, weights=b, base=padded(starts[-1], c["n"], 1.0, _DTYPE[c["out"]]), starts=_ints(starts), starts_host=starts,
                which=which.to(dev), which_host=which.tolist(), scales=torch.rand(c["count"], generator=g, device=dev) + 0.5)


# ---------------------------------------------------------------------------------------- plain forms
def _weights(x):
    """What a row of probabilities weighs, in 64 bits."""
    return torch.nan_to_num(x.double(), nan=0.0, posinf=3.4028234663852886e38, neginf=0.0).clamp(min=0.0)


def _plain_verify(s):
    dev, batch, new = s["tokens"].device, s["b"], s["new"]
    starts = s["starts"].long()
    first, counts = starts[:-1], starts[1:] - starts[:-1]
    each = torch.arange(batch, device=dev)
    node = torch.zeros(batch, dtype=torch.int64, device=dev)
    kept = torch.full((batch, new + 1), -1, dtype=torch.int32, device=dev)
    kept[:, 0] = 0
    many = torch.ones(batch, dtype=torch.int64, device=dev)
    w, mass = _weights(s["target"][first]), torch.ones(batch, dtype=torch.float64, device=dev)
    for i in range(1, new):
        row = (first + i).clamp(max=s["total"] - 1)
        child = (i < counts) & (s["parents"][row].long() == node)
        x = s["tokens"][row]
        wx = w[each, x]
        q = None if s["draft"] is None else _weights(s["draft"][first + node])
        qx = 1.0 if q is None else q[each, x]
        stands = child & (wx > 0) & (s["accept"][row].double() * mass * qx < wx)
        falls = child & ~stands
        if q is None:
            rest = w.clone()
            rest[each, x] = 0.0
            less = (mass - wx).clamp(min=0.0)
        else:
            rest = (w - mass[:, None] * q).clamp(min=0.0)
            less = rest.sum(-1)
        w = torch.where(falls[:, None], rest, torch.where(stands[:, None], _weights(s["target"][row]), w))
        mass = torch.where(falls, less, torch.where(stands, torch.ones_like(mass), mass))
        node = torch.where(stands, i, node)
        kept[each, torch.where(stands, many, new)] = i
        many += stands
    kept = kept[:, :new]
    kept = torch.where(torch.arange(new, device=dev) < many[:, None], kept, -1)
    empty = w.sum(-1) == 0
    w = torch.where(empty[:, None], _weights(s["target"][first + node]), w)
    upto = w.cumsum(-1)
    at = (upto <= (s["sample"].double() * upto[:, -1])[:, None]).sum(-1)
    last = (torch.arange(w.shape[1], device=dev) * (w > 0)).amax(-1)  # (a border that rounding puts behind the last)
    return kept.contiguous(), many.int(), torch.minimum(at, last)


def _places(s):
    """Of every packed row: its position, and the page and row of the page that hold it."""
    row = torch.arange(s["total"], device=s["starts"].device)
    owner = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    position = s["lengths"].long()[owner] + row - s["starts"].long()[owner]
    return s["table"][owner, position // s["page"]].long(), position % s["page"]


def _quantised(x):
    """e4m3 codes and exponents: the scale is the least power of two that brings the row's largest magnitude to 448 or less."""
    x = x.float()
    most = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(most)  # most = mantissa * 2^exponent, 448 = 0.875 * 2^9
    e = (exponent - 9 + (mantissa > 0.875).int() + 127).clamp(1, 254)
    e = torch.where(most == 0, torch.ones_like(e), e)
    return torch.ldexp(x, (127 - e)[..., None]).to(torch.float8_e4m3fn), e.to(torch.uint8)


def _bytes(t):
    """What can be indexed, of tensors that hold 8-bit floats too."""
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _plain_write(s):
    page, at = _places(s)
    for i, x in enumerate((s["k"], s["v"])):
        if len(s["cache"]) == 4:
            code, e = _quantised(x)
            _bytes(s["cache"][i])[page, :, at] = _bytes(code)
            s["cache"][2 + i][page, :, at] = e
        else:
            s["cache"][i][page, :, at] = x


def _plain_keep(s, kept, counts):
    lengths, page = s["lengths"].long(), s["page"]
    i = torch.arange(kept.shape[1], device=kept.device)
    use = i < counts[:, None]
    # (the first node stays where it is: in the place of what is not kept it moves onto itself again)
    come, go = (lengths[:, None] + torch.where(use, x, 0) for x in (kept.long(), i))
    each = torch.arange(len(lengths), device=kept.device)[:, None]
    (p, r), (q, t) = ((s["table"][each, x // page].long(), x % page) for x in (come, go))
    for x in s["cache"]:
        x = _bytes(x)
        x[q, :, t] = x[p, :, r]
    return (lengths + counts).int()


def _plain_fork(s):
    table, lengths, page = s["table"].long(), s["lengths"].long(), s["page"]
    parent = s["parents"].long()
    stays = parent >= 0
    lengths = torch.where(stays, lengths[parent.clamp(min=0)], 0)
    kept = torch.arange(table.shape[1], device=table.device) < (-(-lengths // page))[:, None]
    new = torch.where(stays[:, None] & kept, table[parent.clamp(min=0)], -1)
    users = torch.zeros(len(s["users"]) + 1, dtype=torch.int64, device=table.device)
    for t, sign in ((table, -1), (new, 1)):
        users.index_add_(0, torch.where(t < 0, len(s["users"]), t).flatten(), torch.full((t.numel(),), sign, device=t.device))
    return (s["users"] + users[:-1]).int(), new.int(), lengths.int()


def _plain_grow(s, users, table, lengths):
    dev, page = table.device, s["page"]
    table, users, length = table.long(), users.long(), lengths.long()
    batch, width = table.shape
    counts = (s["starts"][1:] - s["starts"][:-1]).long()
    slot = torch.arange(width, device=dev)
    touched = (slot >= (length // page)[:, None]) & (slot < (-(-(length + counts) // page))[:, None]) & (counts > 0)[:, None]
    absent = touched & (table < 0)
    # a page that others have too is replaced, but for the last that has it
    at = (length // page).clamp(max=width - 1)
    each = torch.arange(batch, device=dev)
    partial = table[each, at]
    writes = touched[each, at] & (partial >= 0)
    before = ((partial[None] == partial[:, None]) & writes[None] & (each[None] < each[:, None])).sum(-1)
    swap = writes & (users[partial.clamp(min=0)] - before > 1)
    absent[each[:, None], at[:, None]] |= swap[:, None]
    need = absent.sum(-1)
    upto = need.cumsum(0)
    free = users == 0
    granted = (upto <= free.sum()) | ((need == 0) & (before == 0))
    take = absent & granted[:, None]
    rank = take.flatten().cumsum(0) - 1
    order = torch.sort((~free).int(), stable=True).indices  # free pages first, lowest first
    page_of = order[rank.clamp(0, len(users) - 1)].view(batch, width)
    new = torch.where(take, page_of, table)
    swap = swap & granted
    users = users.index_add(0, torch.where(swap, partial, 0), -swap.long())
    users = users + torch.zeros_like(users).index_add_(0, torch.where(take, page_of, 0).flatten(), take.flatten().long())
    to = new[each, at]
    for x in s["cache"]:
        x = _bytes(x)
        kept = (torch.arange(page, device=dev) < (length % page)[:, None])
        come, go = torch.where(swap, partial, order[-1]), torch.where(swap, to, order[-1])  # (elsewhere a page that is used, onto itself)
        shape = [batch, 1, page] + [1] * (x.dim() - 3)
        x[go] = torch.where((kept & swap[:, None]).view(shape), x[come], x[go])
    return users.int(), new.int(), torch.where(granted, counts, 0).int()


def _plain_compact(s):
    users, table = s["users"], s["table"].long()
    used = users != 0
    many = used.sum()
    page = torch.arange(len(users), device=users.device)
    hole, mover = ~used & (page < many), used & (page >= many)
    n = len(users)
    # the k-th hole and the k-th that moves
    holes, movers = (torch.sort((~m).int(), stable=True).indices for m in (hole, mover))
    moves = page < mover.sum()
    come, go = torch.where(moves, movers, page[-1:]), torch.where(moves, holes, page[-1:])
    goes = torch.cat((page, page.new_full((1,), -1)))
    goes[torch.where(moves, movers, n)] = torch.where(moves, holes, -1)
    new_users = torch.where(mover, 0, users)
    spread = torch.zeros(n + 1, dtype=users.dtype, device=users.device)
    spread[torch.where(moves, holes, n)] = users[movers]
    new_users = torch.where(hole, spread[:-1], new_users)
    last = moves.view(-1, 1, 1)
    for x in s["cache"]:
        x = _bytes(x)
        for first in range(0, s["moved"], 512):  # (pieces that fit)
            part = slice(first, min(first + 512, n))
            x[go[part]] = torch.where(last[part].view([-1] + [1] * (x.dim() - 1)), x[come[part]], x[go[part]])
    return new_users, torch.where(table < 0, table, goes[table]).int(), many.int().view(1)


def _plain_adapters(s):
    out = s["base"].clone()
    for i, w in enumerate(s["which_host"]):
        if w < 0:
            continue
        rows = slice(s["starts_host"][i], s["starts_host"][i + 1])
        part = (s["x"][rows].float() @ s["a"][w].float().T) @ s["weights"][w].float().T
        out[rows] = (s["base"][rows].float() + s["scales"][w] * part).to(out.dtype)
    return out


def _held(cache):
    """A cache as it stands."""
    return {"pages%d" % i: x for i, x in enumerate(cache)}


def run(state):
    s = state
    kind = s["kind"]
    if own:
        import frisk_b200 as F
    if kind in ("verify", "settle"):
        if own:
            if kind == "settle":
                F.cache_write(s["cache"], s["k"], s["v"], s["table"], s["starts"], s["lengths"])
            kept, counts, token = F.draft_verify(s["tokens"], s["parents"] if s["tree"] else None, s["starts"], s["target"], s["draft"], s["accept"], s["sample"],
                                                 max_new=s["new"])
            if kind == "verify":
                return kept, counts, token
            lengths = F.cache_keep(s["cache"], s["table"], s["starts"], s["lengths"], kept, counts)
        else:
            if kind == "settle":
                _plain_write(s)
            kept, counts, token = _plain_verify(s)
            if kind == "verify":
                return kept, counts, token
            lengths = _plain_keep(s, kept, counts)
        return dict(_held(s["cache"]), kept=kept, counts=counts, token=token, lengths=lengths)
    if kind == "branch":
        if own:
            users, table, lengths = F.cache_fork(s["cache"], s["users"], s["table"], s["lengths"], s["parents"])
            users, table, granted = F.cache_grow(s["cache"], users, table, s["starts"], lengths)
        else:
            users, table, lengths = _plain_fork(s)
            users, table, granted = _plain_grow(s, users, table, lengths)
        return dict(_held(s["cache"]), users=users, table=table, lengths=lengths, granted=granted)
    if kind == "copy":
        if own:
            F.cache_copy(s["cache"], s["source"], s["target"], into=s["into"])
        else:
            for x, y in zip(s["cache"], s["into"]):
                _bytes(y)[s["target"].long()] = _bytes(x)[s["source"].long()]
        return _held(s["into"])
    if kind == "compact":
        users, table, used = F.cache_compact(s["cache"], s["users"], s["table"]) if own else _plain_compact(s)
        return dict(_held(s["cache"]), users=users, table=table, used=used)
    if own:
        return F.adapter_gemm(s["x"], s["a"], s["weights"], s["base"], s["starts"], s["which"], scales=s["scales"])
    return _plain_adapters(s)


# ---------------------------------------------------------------------------------------- what a pass cannot do without
def _token_bytes(c):
    """Keys and values of one token in the cache."""
    return 2 * c["hkv"] * (c["d"] * _SIZE[c["held"]] + (1 if c["held"] == "e4m3" else 0))


def work(case):
    c = case
    if c["kind"] in ("verify", "settle"):
        counts, _ = _ragged(c)
        # every sequence ends with a token drawn from one row of the target's; where a draft is given, with the draft's row taken off it
        values = c["b"] * c["vocab"] * (2 if c["draft"] and c["new"] > 1 else 1)
        total = {"bytes": values * _SIZE[c["dtype"]] + sum(counts) * 16 + 4 * c["b"] * (c["new"] + 3), "flops": 2 * values}
        if c["kind"] == "settle":  # the rows are read and written; half of them are moved
            total["bytes"] += sum(counts) * (2 * c["hkv"] * c["d"] * _SIZE[c["rows"]] + 2 * _token_bytes(c))
        return total
    if c["kind"] == "branch":
        lengths, _ = _group_lengths(c)
        parents, counts = _branch_plan(c)
        width = max(-(-(n + m) // c["page"]) for n, m in zip(lengths, _group_lengths(c)[1])) + 2
        copied = 0  # keys in the last pages that come to be shared: of every holder but one
        for g, n in enumerate(lengths):
            mine = [p for p in parents[g * c["each"]:(g + 1) * c["each"]] if p >= 0]
            copied += (len(mine) - len(set(mine))) * (n % c["page"])
        held = sum(-(-n // c["page"]) for n in lengths)
        return {"bytes": 2 * copied * _token_bytes(c) + 8 * len(parents) * width + 8 * held + 20 * len(parents), "flops": 2 * len(parents) * width}
    if c["kind"] == "copy":
        return {"bytes": c["moved"] * (2 * c["page"] * _token_bytes(c) + 8), "flops": c["moved"]}
    if c["kind"] == "compact":
        moves = c["moved"] * (c["pages"] - c["moved"]) // c["pages"]  # used pages behind the used ones' count, as they are spread evenly
        return {"bytes": 2 * moves * c["page"] * _token_bytes(c) + 8 * c["pages"] + 8 * c["moved"], "flops": c["pages"]}
    counts, _ = _ragged(c)
    rows, e = sum(counts), _SIZE[c["dtype"]]
    return {"bytes": rows * (c["k"] * e + 2 * c["n"] * _SIZE[c["out"]]) + min(c["b"], c["count"]) * c["rank"] * (c["k"] + c["n"]) * e,
            "flops": 2 * rows * c["rank"] * (c["k"] + c["n"])}


# ---------------------------------------------------------------------------------------- in 64 bits, from the definitions
def _exact_verify(s):
    tokens, parents, counts, starts = s["tokens"].tolist(), s["parents"].tolist(), s["counts"], s["starts_host"]
    accept = s["accept"].tolist()
    kept, many, last = torch.full((s["b"], s["new"]), -1, dtype=torch.int32), [], []
    for b, n in enumerate(counts):
        first, node, path = starts[b], 0, [0]
        while True:
            p = s["target"][first + node].double()
            q = None if s["draft"] is None else s["draft"][first + node].double()
            left, chosen = p.clone(), None  # a distribution, up to its sum
            whole = 1.0
            for i in range(node + 1, n):
                if parents[first + i] != node:
                    continue
                x = tokens[first + i]
                here, there = float(left[x]) / whole if whole > 0 else 0.0, 1.0 if q is None else float(q[x])
                if here > 0 and accept[first + i] * there < here:
                    chosen = i
                    break
                if q is None:
                    whole = max(0.0, whole - float(left[x]))
                    left[x] = 0.0
                else:
                    left = torch.relu(left / whole - q)
                    whole = float(left.sum())
            if chosen is None:
                break
            node = chosen
            path.append(node)
        upto = torch.cumsum(left if float(left.sum()) > 0 else p, 0)
        last.append(int(torch.searchsorted(upto, s["sample"][b].double() * upto[-1], right=True).clamp(max=len(p) - 1)))
        kept[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
        many.append(len(path))
    dev = s["tokens"].device
    return kept.to(dev), _ints(many, dev), torch.tensor(last, device=dev)


def _exact_e4m3(x):
    """(code values, exponents): the nearest e4m3 value to x / 2^(e - 127), ties to even."""
    most = x.abs().amax(-1)
    e = torch.ceil(torch.log2(most / 448.0))
    e = torch.where(torch.exp2(e) * 448.0 < most, e + 1, e)
    e = torch.where(torch.exp2(e - 1) * 448.0 >= most, e - 1, e)
    e = torch.where(most > 0, (e + 127).clamp(1, 254), torch.ones_like(e))
    y = x / torch.exp2(e - 127)[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)  # three bits behind the first one
    return torch.round(y / step) * step, e


def _exact_settle(s):
    kept, counts, token = _exact_verify(s)
    cache = [x.double() for x in s["cache"][:2]]
    rows = [_exact_e4m3(x.double())[0] if len(s["cache"]) == 4 else x.double() for x in (s["k"], s["v"])]
    table, page = s["table"].tolist(), s["page"]
    for b, n in enumerate(counts.tolist()):
        path = kept[b].tolist()[:n]
        for i in range(s["counts"][b]):  # a kept row comes from further behind; the others stay as they were written
            row = s["starts_host"][b] + (path[i] if i < n else i)
            at = s["lengths_host"][b] + i
            for x, held in zip(rows, cache):
                held[table[b][at // page], :, at % page] = x[row]
    return dict(_held(cache), kept=kept, counts=counts, token=token, lengths=s["lengths"] + counts)


def _exact_branch(s):
    users, table, lengths, page = s["users"].tolist(), s["table"].tolist(), s["lengths"].tolist(), s["page"]
    starts, width = s["starts"].tolist(), s["width"]
    new, lens = [], []
    for parent in s["parents"].tolist():
        n = lengths[parent] if parent >= 0 else 0
        pages = -(-n // page)
        new.append((table[parent][:pages] if parent >= 0 else []) + [-1] * (width - pages))
        lens.append(n)
    for old, row in zip(table, new):
        for p in old:
            users[p] -= p >= 0
        for p in row:
            users[p] += p >= 0
    cache = [x.double() for x in s["cache"][:2]]
    free = [p for p, n in enumerate(users) if n == 0]
    granted = []
    for b, row in enumerate(new):
        n = starts[b + 1] - starts[b]
        for i in range(lens[b] // page, -(-(lens[b] + n) // page) if n else 0):
            if row[i] >= 0 and users[row[i]] == 1:
                continue
            p = free.pop(0)  # (there are enough in these cases)
            if row[i] >= 0:
                for x in cache:
                    x[p, :, :lens[b] % page] = x[row[i], :, :lens[b] % page]
                users[row[i]] -= 1
            users[p] = 1
            row[i] = p
        granted.append(n)
    return dict(_held(cache), users=_ints(users), table=_ints(new), lengths=_ints(lens), granted=_ints(granted))


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "verify":
        return _exact_verify(s)
    if kind == "settle":
        return _exact_settle(s)
    if kind == "branch":
        return _exact_branch(s)
    if kind == "copy":
        into = [x.double() for x in s["into"][:2]]
        for x, y in zip(s["cache"], into):
            y.index_copy_(0, s["target"].long(), _bytes(x).index_select(0, s["source"].long()).view(x.dtype).double())
        return _held(into)
    if kind == "compact":
        users, table = s["users"].tolist(), s["table"].tolist()
        used = [p for p, n in enumerate(users) if n]
        holes = [p for p in range(len(used)) if not users[p]]
        goes = dict(zip([p for p in used if p >= len(used)], holes))
        cache = [x.double() for x in s["cache"][:2]]
        if goes:
            come, go = (torch.tensor(list(x), device=cache[0].device) for x in (goes.keys(), goes.values()))
            for x in cache:
                x.index_copy_(0, go, x.index_select(0, come))
        for p, to in goes.items():
            users[to], users[p] = users[p], 0
        return dict(_held(cache), users=_ints(users), table=_ints([[goes.get(p, p) for p in row] for row in table]), used=_ints([len(used)]))
    out = s["base"].double()
    for i, w in enumerate(s["which_host"]):
        if w >= 0:
            lo, hi = s["starts_host"][i], s["starts_host"][i + 1]
            rank = torch.einsum("rk,mk->rm", s["x"][lo:hi].double(), s["a"][w].double())
            out[lo:hi] += float(s["scales"][w]) * torch.einsum("rm,nm->rn", rank, s["weights"][w].double())
    return out
