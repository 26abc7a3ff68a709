"""Performance cases of the paged key/value cache and what goes through it.

Four operators: ``rotary`` (with its backward), ``cache_write``, ``cache_read`` and ``cache_attention``.  A case names its kind:

* ``rotary``     rotary positions on the queries and keys of N tokens
* ``rotary_bwd`` the gradients of the same
* ``store``      new tokens written into the pages, and those tokens read back as the cache holds them
* ``read``       whole sequences gathered out of the pages into packed rows
* ``attend``     the attention of drafted tokens over the cache (one token a sequence, a chain, or a tree with its mask)
* ``step``       one step of a server: rotate, write, attend

Packed rows: sequence b's new tokens are rows starts[b] .. starts[b + 1] - 1, and lengths[b] keys of it are in the cache before them.
A cache is (k, v) of [pages, heads, page, D], with an 8-bit exponent for every token and head where it holds 8-bit floats.
"""
import math
import random

import torch

own = False

_DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
_SIZE = {"fp16": 2, "bf16": 2, "fp32": 4, "e4m3": 1}


def _rotary(n, h, hkv, d, dim, dtype, interleaved, far, scaling="none", kind="rotary", **name):
    return dict(name, kind=kind, n=n, h=h, hkv=hkv, d=d, dim=dim, dtype=dtype, interleaved=interleaved, far=far, scaling=scaling)


def _cache(kind, b, new, length, hkv, group, d, page, dtype, held, tree="none", **name):
    """``new`` tokens and up to ``length`` keys in the cache for each of ``b`` sequences; ``held``: the cache's element type."""
    return dict(name, kind=kind, b=b, new=new, length=length, hkv=hkv, group=group, d=d, page=page, dtype=dtype, held=held, tree=tree)


def listed():
    return [
        # the queries and keys of a batch of 32 that decodes: the smallest call, all latency
        _rotary(32, 32, 8, 128, 128, "bf16", False, 131072, name="rotary_decode"),
        # a prompt of 8192 tokens at positions beyond the trained ones, pairs side by side
        _rotary(8192, 32, 8, 128, 128, "bf16", True, 131072, "yarn", name="rotary_prompt_yarn"),
        # training: gradients of a ragged count of tokens, half of each head rotated, heads of 80
        _rotary(4099, 20, 20, 80, 40, "fp32", False, 4096, "linear", kind="rotary_bwd", name="rotary_backward_part"),
        # one decoded token for each of 64 sequences into an 8-bit cache
        _cache("store", 64, 1, 2000, 8, 4, 128, 16, "bf16", "e4m3", name="store_decode_e4m3"),
        # prompts of eight ragged sequences, 16 thousand tokens at most, quantised as they are written
        _cache("store", 8, 2048, 0, 8, 4, 128, 64, "bf16", "e4m3", name="store_prompts_e4m3"),
        # long sequences gathered out of a 16-bit cache for a dense pass over them
        _cache("read", 4, 16000, 0, 8, 4, 128, 32, "bf16", "bf16", name="read_bf16"),
        # the same out of an 8-bit cache, heads of 64
        _cache("read", 7, 9001, 0, 4, 4, 64, 16, "fp16", "e4m3", name="read_e4m3"),
        # a single sequence that decodes, short: all latency
        _cache("attend", 1, 1, 200, 8, 4, 128, 16, "bf16", "bf16", name="attend_one_short"),
        # a batch that decodes: 32 query heads over 8 key heads, caches of up to 8000 keys
        _cache("attend", 32, 1, 8000, 8, 4, 128, 64, "bf16", "bf16", name="attend_decode"),
        # trees of 24 drafted tokens over an 8-bit cache
        _cache("attend", 16, 24, 6000, 8, 4, 128, 64, "bf16", "e4m3", "tree", name="attend_tree_e4m3"),
        # trees of 64 drafted tokens over long 16-bit caches
        _cache("attend", 8, 64, 32000, 8, 8, 128, 128, "bf16", "bf16", "tree", name="attend_tree_long"),
        # one step of a server: 5 drafted tokens a sequence, heads of 64, 8-bit cache
        _cache("step", 24, 5, 3000, 4, 8, 64, 32, "fp16", "e4m3", "tree", name="step_tree_e4m3"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary_bwd", "store", "read", "attend", "attend", "attend", "attend", "step"])
    if kind in ("rotary", "rotary_bwd"):
        hkv = rng.choice([1, 2, 4, 8, 20])
        h = hkv * rng.choice([1, 4, 8]) if hkv < 20 else 20
        d = rng.choice([64, 80, 96, 128, 128, 256])
        return _rotary(_log(rng, 1, 8192), h, hkv, d, rng.choice([d, d, d // 2]), rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                       rng.random() < 0.5, _log(rng, 4096, 1 << 20), rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]), kind)
    held = rng.choice(["e4m3", "16"])
    dtype = rng.choice(["bf16", "fp16"])
    held = dtype if held == "16" else held
    hkv, group, d, page = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    if kind == "store":
        new = _log(rng, 1, 2048)
        return _cache(kind, _log(rng, 1, max(1, 16384 // new)) if new > 16 else _log(rng, 1, 128), new, _log(rng, 1, 2000), hkv, group, d, page, dtype, held)
    if kind == "read":
        b = _log(rng, 1, 16)
        return _cache(kind, b, _log(rng, 1, 64000 // b), 0, hkv, group, d, page, dtype, held)
    b, new = _log(rng, 1, 64), rng.choice([1, 1, _log(rng, 1, 64), _log(rng, 1, 64)])
    if kind == "step":
        return _cache(kind, b, new, _log(rng, 1, 4000), hkv, group, d, page, dtype, held, "tree" if new > 1 else "none")
    return _cache(kind, b, new, _log(rng, 1, min(32000, 256000 // b)), hkv, group, d, page, dtype, held, rng.choice(["tree", "tree", "none"]) if new > 1 else "none")


# ---------------------------------------------------------------------------------------- frequencies
def _frequencies(dim, scaling):
    """(radians per position of each pair in 64 bits, factor on the rotated values).  Contexts 8 times the trained 4096."""
    base, factor, trained = 10000.0, 8.0, 4096
    if scaling == "ntk":  # a larger base: the slowest pair turns `factor` times slower
        base *= factor ** (dim / max(1, dim - 2))
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":  # pairs that turn more than 32 times over the trained context stay, those under once are stretched
        at = [trained * x / (2 * math.pi) for x in f]
        keep = [min(1.0, max(0.0, (t - 1.0) / (32.0 - 1.0))) for t in at]
        f = [x * (r + (1 - r) / factor) for x, r in zip(f, keep)]
    if scaling == "wavelength":  # the same between 1 and 4 turns, and no factor on the values
        at = [trained * x / (2 * math.pi) for x in f]
        keep = [min(1.0, max(0.0, (t - 1.0) / (4.0 - 1.0))) for t in at]
        f = [x * (r + (1 - r) / factor) for x, r in zip(f, keep)]
    return f, 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0


# ---------------------------------------------------------------------------------------- inputs
def _tree_mask(gen, total, starts, new):
    """bool [total, new]: token i sees itself and its ancestors; the parent of token i > 0 is one of the up to 8 tokens before it."""
    mask = torch.zeros(total, new, dtype=torch.bool)
    for s, e in zip(starts[:-1], starts[1:]):
        back = torch.randint(1, 9, (e - s,), generator=gen).tolist()
        for i in range(e - s):
            if i:
                mask[s + i] = mask[s + max(0, i - back[i])]
            mask[s + i, i] = True
    return mask


def _ragged(c):
    """The new tokens and the cached keys of every sequence: between two thirds and all of the largest count, by the case alone."""
    if c["b"] == 1:
        return [c["new"]], [c["length"]]
    rng = random.Random(c["b"] * 1000003 + c["new"] * 1009 + c["length"])
    counts = [rng.randint(max(1, 2 * c["new"] // 3), c["new"]) for _ in range(c["b"])]
    return counts, [rng.randint(2 * c["length"] // 3, c["length"]) for _ in range(c["b"])]


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    c, dt = dict(case), _DTYPE[case["dtype"]]
    if c["kind"].startswith("rotary"):
        # one buffer of projected rows, as a fused projection leaves them: queries, keys (and values, untouched)
        rows = torch.randn(c["n"], (c["h"] + 2 * c["hkv"]) * c["d"], generator=g, device=dev).to(dt)
        q = rows[:, :c["h"] * c["d"]].view(c["n"], c["h"], c["d"])
        k = rows[:, c["h"] * c["d"]:(c["h"] + c["hkv"]) * c["d"]].view(c["n"], c["hkv"], c["d"])
        first = int(torch.randint(0, max(1, c["far"] - c["n"]), (1,), generator=gen))
        positions = (torch.arange(c["n"]) + first).to(dev) if c["n"] > 64 else torch.randint(0, c["far"], (c["n"],), generator=gen).to(dev)
        f, amplitude = _frequencies(c["dim"], c["scaling"])
        return dict(c, q=q, k=k, positions=positions, frequencies=torch.tensor(f, dtype=torch.float64, device=dev), amplitude=amplitude)
    b, new, page, d, hkv = c["b"], c["new"], c["page"], c["d"], c["hkv"]
    counts, lengths = _ragged(c)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    total = starts[-1]
    need = [-(-(n + m) // page) for n, m in zip(lengths, counts)]
    pages = sum(need) + 8
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.zeros(b, max(need), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    shape = (pages, hkv, page, d)
    if c["held"] == "e4m3":
        def values():
            return torch.randn(shape, generator=g, device=dev, dtype=torch.float16).mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)

        def exponents():
            return torch.randint(117, 121, shape[:3], generator=g, device=dev, dtype=torch.uint8)
        cache = values(), values(), exponents(), exponents()
    else:
        cache = torch.randn(shape, generator=g, device=dev, dtype=dt), torch.randn(shape, generator=g, device=dev, dtype=dt)
    # the rows of a fused projection: queries, keys, values
    h = hkv * c["group"]
    rows = torch.randn(total, (h + 2 * hkv) * d, generator=g, device=dev).to(dt)
    q = rows[:, :h * d].view(total, h, d)
    k, v = (rows[:, (h + i * hkv) * d:(h + (i + 1) * hkv) * d].view(total, hkv, d) for i in (0, 1))
    state = dict(c, cache=cache, q=q, k=k, v=v, table=table.to(dev), total=total, max_new=max(counts),
                 starts=torch.tensor(starts, dtype=torch.int32, device=dev), lengths=torch.tensor(lengths, dtype=torch.int32, device=dev))
    mask = _tree_mask(gen, total, starts, max(counts)) if c["tree"] == "tree" else None
    state["mask"] = None if mask is None else mask.to(dev)
    if c["kind"] == "step":
        depth = mask.sum(1) - 1 if mask is not None else torch.tensor([i for n in counts for i in range(n)])
        owner = torch.tensor([i for i, n in enumerate(counts) for _ in range(n)])
        state["positions"] = (torch.tensor(lengths)[owner] + depth).to(dev)
        f, state["amplitude"] = _frequencies(d, "none")
        state["frequencies"] = torch.tensor(f, dtype=torch.float64, device=dev)
    return state


# ---------------------------------------------------------------------------------------- plain forms
def _plain_rotary(x, positions, frequencies, amplitude, interleaved, sign):
    dim = 2 * frequencies.numel()
    angle = positions.double()[:, None] * frequencies
    cos, sin = (amplitude * angle.cos()).float()[:, None], (sign * amplitude * angle.sin()).float()[:, None]
    r = x[..., :dim].float()
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :dim // 2], r[..., dim // 2:])
    pair = (a * cos - b * sin, b * cos + a * sin)
    r = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat((r.to(x.dtype), x[..., dim:]), -1)


def _places(s):
    """Of every packed row: its sequence, its position, and the page and row of the page that hold it."""
    row = torch.arange(s["total"], device=s["starts"].device)
    owner = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    position = s["lengths"].long()[owner] + row - s["starts"].long()[owner]
    return owner, position, s["table"][owner, position // s["page"]].long(), position % s["page"]


def _quantised(x):
    """e4m3 codes and exponents: the scale is the least power of two that brings the row's largest magnitude to 448 or less."""
    x = x.float()
    most = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(most)  # most = mantissa * 2^exponent, 448 = 0.875 * 2^9
    e = (exponent - 9 + (mantissa > 0.875).int() + 127).clamp(1, 254)
    e = torch.where(most == 0, torch.ones_like(e), e)
    return torch.ldexp(x, (127 - e)[..., None]).to(torch.float8_e4m3fn), e.to(torch.uint8)


def _plain_write(s, k, v):
    _, _, page, at = _places(s)
    cache = s["cache"]
    for i, x in enumerate((k, v)):
        if len(cache) == 4:
            code, e = _quantised(x)
            cache[i].view(torch.uint8)[page, :, at] = code.view(torch.uint8)
            cache[2 + i][page, :, at] = e
        else:
            cache[i][page, :, at] = x


def _values(cache, i, page, at):
    x = cache[i].view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn) if len(cache) == 4 else cache[i][page, :, at]
    x = x.float()
    return torch.ldexp(x, cache[2 + i][page, :, at].int()[..., None] - 127) if len(cache) == 4 else x


def _plain_read(s):
    _, _, page, at = _places(s)
    return tuple(_values(s["cache"], i, page, at).to(s["k"].dtype) for i in (0, 1))


def _plain_attend(s, q):
    dev, b = q.device, s["b"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    counts = starts[1:] - starts[:-1]
    new, keys = s["max_new"], s["table"].shape[1] * s["page"]
    # padded to [sequence, new token] and [sequence, key]
    i = torch.arange(new, device=dev)
    row = (starts[:-1, None] + i).clamp(max=s["total"] - 1)
    j = torch.arange(keys, device=dev)
    page, at = s["table"][:, j // s["page"]].long(), (j % s["page"]).expand(b, -1)
    k, v = (_values(s["cache"], n, page, at) for n in (0, 1))  # [sequence, key, head, D]
    x = q[row].float().view(b, new, s["hkv"], s["group"], s["d"])
    score = torch.einsum("bihgd,bjhd->bhgij", x, k) * s["d"] ** -0.5
    ahead = j[None] - lengths[:, None]  # which new token a key is, negative for those before
    if s["mask"] is None:
        seen = ahead[:, None] <= i[None, :, None]
    else:
        width = s["mask"].shape[1]
        drafted = torch.gather(s["mask"][row], 2, ahead.clamp(0, width - 1)[:, None].expand(b, new, keys))
        seen = (ahead < 0)[:, None] | (drafted & (ahead < torch.minimum(counts, torch.tensor(width, device=dev))[:, None])[:, None])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    p = (score - most.masked_fill(most == -math.inf, 0.0)).exp()
    total = p.sum(-1)
    v = v.masked_fill((ahead >= counts[:, None])[:, :, None, None], 0.0)
    o = torch.einsum("bhgij,bjhd->bihgd", p, v) / total.masked_fill(total == 0, 1.0).permute(0, 3, 1, 2)[..., None]
    return o.reshape(b, new, -1, s["d"])[i[None] < counts[:, None]].to(q.dtype)


def _held(s):
    """The cache as it stands."""
    return {"pages%d" % i: x for i, x in enumerate(s["cache"])}


def run(state):
    s = state
    kind = s["kind"]
    if own:
        import frisk_b200 as F
    if kind in ("rotary", "rotary_bwd"):
        sign = 1.0 if kind == "rotary" else -1.0
        if own:
            turn = F.rotary if kind == "rotary" else F.rotary_backward
            return turn(s["q"], s["k"], s["positions"], s["frequencies"], amplitude=s["amplitude"], interleaved=s["interleaved"])
        return tuple(_plain_rotary(x, s["positions"], s["frequencies"], s["amplitude"], s["interleaved"], sign) for x in (s["q"], s["k"]))
    if kind == "store":
        if own:
            F.cache_write(s["cache"], s["k"], s["v"], s["table"], s["starts"], s["lengths"])
            back = F.cache_read(s["cache"], s["table"], s["starts"], s["lengths"], s["total"], dtype=s["k"].dtype)
        else:
            _plain_write(s, s["k"], s["v"])
            back = _plain_read(s)
        return dict(_held(s), k=back[0], v=back[1])
    if kind == "read":
        if own:
            return F.cache_read(s["cache"], s["table"], s["starts"], s["lengths"], s["total"], dtype=s["k"].dtype)
        return _plain_read(s)
    if kind == "attend":
        if own:
            return F.cache_attention(s["cache"], s["q"], s["table"], s["starts"], s["lengths"], mask=s["mask"], max_new=s["max_new"])
        return _plain_attend(s, s["q"])
    if own:
        q, k = F.rotary(s["q"], s["k"], s["positions"], s["frequencies"], amplitude=s["amplitude"])
        F.cache_write(s["cache"], k, s["v"], s["table"], s["starts"], s["lengths"])
        out = F.cache_attention(s["cache"], q, s["table"], s["starts"], s["lengths"], mask=s["mask"], max_new=s["max_new"])
    else:
        q, k = (_plain_rotary(x, s["positions"], s["frequencies"], s["amplitude"], False, 1.0) for x in (s["q"], s["k"]))
        _plain_write(s, k, s["v"])
        out = _plain_attend(s, q)
    return dict(_held(s), out=out)


# ---------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    e = _SIZE[c["dtype"]]
    if c["kind"].startswith("rotary"):
        values = c["n"] * (c["h"] + c["hkv"]) * c["d"]
        return {"bytes": 2 * e * values + 8 * c["n"] + 4 * c["dim"], "flops": 3 * c["n"] * (c["h"] + c["hkv"]) * c["dim"]}
    counts, lengths = _ragged(c)
    new = sum(counts)
    row = 2 * c["hkv"] * (c["d"] * _SIZE[c["held"]] + (1 if c["held"] == "e4m3" else 0))  # of one token in the cache, keys and values
    rows = 2 * c["hkv"] * c["d"] * e                                                      # of one token outside it
    h = c["hkv"] * c["group"]
    if c["kind"] == "store":
        return {"bytes": new * (2 * rows + 2 * row), "flops": 4 * new * c["hkv"] * c["d"]}
    if c["kind"] == "read":
        return {"bytes": new * (rows + row), "flops": 2 * new * c["hkv"] * c["d"]}
    keys = sum(lengths) + new
    bytes_ = keys * row + 2 * new * h * c["d"] * e + (new * c["new"] if c["tree"] == "tree" else 0)
    flops = 4 * sum(n * (m + n) for n, m in zip(counts, lengths)) * h * c["d"]
    if c["kind"] == "step":  # the queries are rotated, the new keys and values written before that
        bytes_ += 2 * new * h * c["d"] * e + new * (3 * rows / 2 + row)
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------------------- in 64 bits, from the definitions
def _exact_rotary(x, positions, f, amplitude, interleaved, sign):
    x = x.double()
    y = x.clone()
    for i in range(f.numel()):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + f.numel())
        t = positions.double() * f[i]
        c, s = amplitude * torch.cos(t)[:, None], sign * amplitude * torch.sin(t)[:, None]
        y[..., a] = c * x[..., a] - s * x[..., b]
        y[..., b] = s * x[..., a] + c * x[..., b]
    return y


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


def _exact_store(s, k, v):
    """The cache after the write, and the written rows as it holds them, sequence by sequence."""
    starts, lengths, page = s["starts"].tolist(), s["lengths"].tolist(), s["page"]
    e4m3 = len(s["cache"]) == 4
    held = [x.double() for x in s["cache"]]
    back = []
    for n, x in enumerate((k, v)):
        code, e = _exact_e4m3(x) if e4m3 else (x, None)
        back.append(code * torch.exp2(e - 127)[..., None] if e4m3 else code)
        for b in range(s["b"]):
            for first in range(starts[b], starts[b + 1], page):
                rows = torch.arange(first, min(first + page, starts[b + 1]), device=x.device)
                at = rows - starts[b] + lengths[b]
                where = s["table"][b].long()[at // page]
                held[n][where, :, at % page] = code[rows]
                if e4m3:
                    held[2 + n][where, :, at % page] = e[rows]
    return held, back


def _exact_attend(s, q, held):
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for b in range(s["b"]):
        n, length = starts[b + 1] - starts[b], lengths[b]
        j = torch.arange(length + n, device=q.device)
        where, at = s["table"][b].long()[j // s["page"]], j % s["page"]
        seen = torch.ones(n, length + n, dtype=torch.bool, device=q.device)
        seen[:, length:] = torch.ones(n, n, device=q.device).tril().bool() if s["mask"] is None else s["mask"][starts[b]:starts[b + 1], :n]
        for h in range(s["hkv"]):
            k, v = (held[i][where, h, at] for i in (0, 1))
            if len(held) == 4:
                k, v = (x * torch.exp2(held[2 + i][where, h, at] - 127)[:, None] for i, x in enumerate((k, v)))
            heads = slice(h * s["group"], (h + 1) * s["group"])
            x = q[starts[b]:starts[b + 1], heads].transpose(0, 1)
            p = torch.softmax((x @ k.T / math.sqrt(s["d"])).masked_fill(~seen, -math.inf), -1)
            out[starts[b]:starts[b + 1], heads] = (p @ v).transpose(0, 1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind in ("rotary", "rotary_bwd"):
        sign = 1.0 if kind == "rotary" else -1.0
        return tuple(_exact_rotary(x, s["positions"], s["frequencies"], s["amplitude"], s["interleaved"], sign) for x in (s["q"], s["k"]))
    if kind == "store":
        held, back = _exact_store(s, s["k"].double(), s["v"].double())
        return dict({"pages%d" % i: x for i, x in enumerate(held[:2])}, k=back[0], v=back[1])
    if kind == "read":
        starts, lengths, page = s["starts"].tolist(), s["lengths"].tolist(), s["page"]
        got = []
        for i in (0, 1):
            part = []
            for b in range(s["b"]):
                j = torch.arange(lengths[b], lengths[b] + starts[b + 1] - starts[b], device=s["table"].device)
                where = s["table"][b].long()[j // page]
                x = s["cache"][i].view(torch.uint8)[where, :, j % page].view(torch.float8_e4m3fn) if len(s["cache"]) == 4 else s["cache"][i][where, :, j % page]
                x = x.double()
                part.append(x * torch.exp2(s["cache"][2 + i][where, :, j % page].double() - 127)[..., None] if len(s["cache"]) == 4 else x)
            got.append(torch.cat(part))
        return tuple(got)
    if kind == "attend":
        return _exact_attend(s, s["q"].double(), [x.double() for x in s["cache"]])
    # what the step rounds on its way (rotated rows to 16 bits, the cache to its type) is part of what it returns and reads
    q, k = (_exact_rotary(x, s["positions"], s["frequencies"], s["amplitude"], False, 1.0).to(x.dtype).double() for x in (s["q"], s["k"]))
    held, _ = _exact_store(s, k, s["v"].double())
    return {"out": _exact_attend(s, q, held)}
