"""Rotary positions, the paged cache and attention over it in 64 bits, element by element from their definitions (CPU tensors)."""
import math

import torch

H = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative to the value


def rotary(x, positions, frequencies, amplitude=1.0, interleaved=False, inverse=False):
    x, y = x.double(), x.double().clone()
    half = len(frequencies)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        t = positions.double() * float(frequencies[i]) * (-1.0 if inverse else 1.0)
        c, s = amplitude * torch.cos(t)[:, None], amplitude * torch.sin(t)[:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def _e4m3_values():
    """Of every code 0 .. 127: 3 fraction bits, 4 exponent bits with bias 7; the last is NaN."""
    out = []
    for code in range(127):
        e, f = code >> 3, code & 7
        out.append((8 + f) * 2.0 ** (e - 10) if e else f * 2.0 ** -9)
    return torch.tensor(out, dtype=torch.float64)


E4M3 = _e4m3_values()


def quantise(x):
    """(codes uint8, exponents uint8) of rows of D elements."""
    x = x.double()
    flat = x.reshape(-1, x.shape[-1])
    codes, exps = torch.zeros(flat.shape, dtype=torch.uint8), torch.zeros(len(flat), dtype=torch.uint8)
    between = (E4M3[1:] + E4M3[:-1]) / 2
    for r, row in enumerate(flat):
        if not torch.isfinite(row).all():
            exps[r] = 255
            continue
        most, e = row.abs().max().item(), 1
        if most > 0:
            e = max(1, math.frexp(most)[1] + 127 - 20)
            while most > 448.0 * 2.0 ** (e - 127):
                e += 1
        y = row.abs() * 2.0 ** (127 - e)
        low = torch.searchsorted(between, y)                      # values below this border
        tie = (low < len(between)) & (between[low.clamp(max=len(between) - 1)] == y) & (low % 2 == 1)
        code = low + tie.long()
        codes[r] = (code + 128 * (torch.signbit(row)).long()).to(torch.uint8)
        exps[r] = e
    return codes.reshape(x.shape), exps.reshape(x.shape[:-1])


def values(cache, which):
    """The cache's keys (0) or values (1) in 64 bits."""
    if len(cache) == 2:
        return cache[which].double()
    codes, e = cache[which].view(torch.uint8).long(), cache[2 + which].double()
    x = torch.cat((E4M3, torch.tensor([math.nan], dtype=torch.float64)))[codes & 127]
    x = torch.where(codes >= 128, -x, x) * torch.exp2(e - 127)[..., None]
    return torch.where((e == 255)[..., None], math.nan, x)


def slots(table, starts, lengths, page):
    """(row, sequence, page, offset) of every packed row that has a place."""
    for b in range(len(lengths)):
        for r in range(int(starts[b]), int(starts[b + 1])):
            pos = int(lengths[b]) + r - int(starts[b])
            yield r, b, int(table[b, pos // page]), pos % page


def write(cache, k, v, table, starts, lengths):
    """A copy of the cache with the rows written."""
    new = [t.clone() for t in cache]
    for which, x in enumerate((k, v)):
        code, e = quantise(x) if len(cache) == 4 else (x, None)
        for r, _, page, at in slots(table, starts, lengths, cache[0].shape[2]):
            if e is None:
                new[which][page, :, at] = code[r]
            else:
                new[which].view(torch.uint8)[page, :, at] = code[r]
                new[2 + which][page, :, at] = e[r]
    return tuple(new)


def seen(rows, length, mask, first):
    """bool [rows, length + rows]: what the new tokens of a sequence see."""
    see = torch.ones(rows, length + rows, dtype=torch.bool)
    if mask is None:
        see[:, length:] = torch.ones(rows, rows).tril().bool()
    else:
        see[:, length:] = False
        w = min(rows, mask.shape[1])
        see[:, length:length + w] = mask[first:first + rows, :w]
    return see


def attention(cache, q, table, starts, lengths, mask=None, scale=None, terms=False):
    """(results, bound): float64 [rows, heads, D], and for each how far a kernel may be off that rounds each probability (and scale
    times probability) by half a step of its operands' type, works in 32 bits otherwise and rounds the result once.

    ``terms``: an 8-bit cache whose products take sums of 8-bit values.  A weight becomes a half and the half three e5m2 values for bf16 (each
    keeps 3 bits of the rest, the last is rounded: off by 2^-9) or four for fp16 (exact), and in either case is off by half of the smallest
    step, 2^-17.  The largest weight times scale stands at 2^12.75 or more, but for the 2^5 that the scales of a tile's values may be apart:
    2^(5 - 17 - 12.75) of it.  A query's e4m3 terms leave 2^-10 of a row scaled to 128 or more."""
    n, heads_q, d = q.shape
    heads, page = cache[0].shape[1], cache[0].shape[2]
    group, scale = heads_q // heads, d ** -0.5 if scale is None else scale
    k_all, v_all = values(cache, 0), values(cache, 1)
    h_out = H[q.dtype]
    h_p = (2.0 ** -9 if q.dtype == torch.bfloat16 else 0.0) + 2.0 ** -11 if terms else H[torch.float16] if len(cache) == 4 else h_out
    out, bound = torch.zeros(n, heads_q, d, dtype=torch.float64), torch.zeros(n, heads_q, d, dtype=torch.float64)
    for b in range(len(lengths)):
        first, rows, length = int(starts[b]), int(starts[b + 1]) - int(starts[b]), int(lengths[b])
        if rows == 0:
            continue
        j = torch.arange(length + rows)
        at = table[b].long()[j // page]
        see = seen(rows, length, mask, first)
        for h in range(heads_q):
            k, v = k_all[at, h // group, j % page], v_all[at, h // group, j % page]
            x = q[first:first + rows, h].double()
            s = (x @ k.T) * scale
            # a key that no row sees may hold anything; one that some rows do not see, too
            s = torch.where(see, s, -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
            total = p.sum(1, keepdim=True)
            p = torch.where(total == 0, 0.0, p / total)
            weighted = torch.where(see[:, :, None], p[:, :, None] * v[None], 0.0)
            o, a = weighted.sum(1), weighted.abs().sum(1)
            # scores: D products summed in 32 bits (2^-23 each, the tensor core may truncate), the exponential 2^-22 and its argument's
            # rounding; they enter numerator and denominator
            kk = torch.where(torch.isfinite(k), k, 0.0)
            mag = (x.abs() @ kk.abs().T).amax(1, keepdim=True) * abs(scale)
            delta = 2 * (d * 2.0 ** -23 * mag + 2.0 ** -22 + 2.0 ** -22 * mag) + (length + rows) * 2.0 ** -24
            if terms:
                delta = delta + 2 * 2.0 ** -17 * x.abs().amax(1, keepdim=True) * kk.abs().sum(1).amax() * abs(scale)
            out[first:first + rows, h] = o
            # (what underflows beside the largest weight: 2^-24 of its step for each key; infinities and NaN have columns of their own)
            far = torch.where(torch.isfinite(weighted), weighted, 0.0).abs().amax(dim=(1, 2))[:, None] * 2.0 ** -22
            if terms:
                e = cache[3][at, h // group, j % page].double()
                scale_v = torch.where(see.any(0) & (e < 255), torch.exp2(e - 127), 0.0)
                codes = torch.where(torch.isfinite(v), v, 0.0).abs() * torch.where(scale_v > 0, 1 / scale_v, 0.0)[:, None]
                far = far + 2.0 ** -24.75 * (p.nan_to_num() * scale_v).amax(1, keepdim=True) * codes.sum(0)[None]
            bound[first:first + rows, h] = h_p * a + delta * a + h_out * (o.abs() + (h_p + delta) * a) + far + 1e-30
    return out, bound
