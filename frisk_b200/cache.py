"""A paged key/value cache: ``paged_cache``, ``cache_write``, ``cache_read`` and ``cache_attention``.

A cache is a tuple of tensors: keys and values [pages, heads, page, D] in float16 or bfloat16, or in float8_e4m3fn with two more
tensors of uint8 [pages, heads, page], the exponents of keys and values; a value is then code * 2 ** (exponent - 127).

A call works on packed rows, the new tokens of a batch one sequence behind the other: rows ``starts[b]`` .. ``starts[b + 1] - 1``
belong to sequence b and sit behind the ``lengths[b]`` keys it has already, so row ``starts[b] + i`` has position ``lengths[b] + i``.
``table[b, i]`` is the page of positions ``i * page`` .. of sequence b.  The three are int32 tensors on the device, so that a captured
step can be replayed with other contents.  Their contents are checked by the kernels: what is out of range is left out, and
``cache_check`` raises.  Rows before ``starts[0]`` and from ``starts[-1]`` on belong to no sequence and are left as they are.
"""
import contextlib

from . import calls, capi
from .calls import context_for
from .execute import _stream_ptr, _torch

_CODES = _BYTE = _INT = None


def _codes():
    global _CODES, _BYTE, _INT
    if _CODES is None:
        torch = _torch()
        _BYTE, _INT = torch.uint8, torch.int32
        _CODES = {torch.float16: capi.F16, torch.bfloat16: capi.BF16, torch.float8_e4m3fn: capi.E4M3}
    return _CODES


def _stream_of(stream, dev):
    torch = _torch()
    if stream is None:
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        return raw(dev) if raw is not None else torch.cuda.current_stream(dev).cuda_stream
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _on_stream(stream, device):
    """What is allocated in it belongs to the stream the kernels run on."""
    if stream is None:
        return contextlib.nullcontext()
    torch = _torch()
    return torch.cuda.stream(stream if hasattr(stream, "cuda_stream") else torch.cuda.ExternalStream(int(stream), device=device))


def _new_like(t):
    """A dense new tensor of the shape, type and device of ``t``."""
    torch = _torch()
    return torch.empty_like(t, memory_format=torch.contiguous_format)


_shapes = {}


def _workspace(nbytes, dev):
    """New scratch of the call's own, so that calls on other streams and captured graphs share none.  (What is kept is a tensor of that
    shape over a single byte: an allocation after its like costs half of one by its size.)"""
    torch = _torch()
    like = _shapes.get((nbytes, dev))
    if like is None:
        like = _shapes[nbytes, dev] = torch.empty(1, dtype=torch.uint8, device=torch.device("cuda", dev)).expand(nbytes)
    return torch.empty_like(like, memory_format=torch.contiguous_format)


def _refuse(what):
    raise ValueError("frisk-b200-cache: " + what)


def paged_cache(pages, heads, page, d, dtype, device="cuda"):
    """A new cache of ``pages`` pages of ``page`` tokens (a power of two from 16 to 1024) with heads of 64 or 128 elements."""
    torch = _torch()
    if dtype not in _codes():
        _refuse("a cache holds float16, bfloat16 or float8_e4m3fn")
    if pages < 1 or heads < 1 or page < 16 or page > 1024 or page & (page - 1) or d not in (64, 128):
        _refuse("sizes outside the contract")
    held = tuple(torch.zeros(pages, heads, page, d, dtype=dtype, device=device) for _ in range(2))
    if dtype != torch.float8_e4m3fn:
        return held
    return held + tuple(torch.zeros(pages, heads, page, dtype=torch.uint8, device=device) for _ in range(2))


def _describe(cache, table, starts, lengths, rows):
    """(descriptor, element code, device index, key heads, D), checked."""
    codes = _CODES or _codes()
    parts = len(cache)
    if parts == 2:
        k, v = cache
        ek = ev = None
    elif parts == 4:
        k, v, ek, ev = cache
    else:
        _refuse("a cache is (k, v), or (k, v, k exponents, v exponents)")
    dtype, shape, dev = k.dtype, k.shape, k.get_device()
    code = codes.get(dtype)
    if code is None or (code == capi.E4M3) != (parts == 4):
        _refuse("a cache holds float16, bfloat16, or float8_e4m3fn with exponents")
    if len(shape) != 4 or v.shape != shape or v.dtype != dtype or not k.is_contiguous() or not v.is_contiguous():
        _refuse("keys and values must be dense [pages, heads, page, D] of one type")
    if dev < 0 or v.get_device() != dev:
        _refuse("tensors must be on one CUDA device (there is no CPU path)")
    pages, heads, page, d = shape
    if parts == 4:
        want = shape[:3]
        for e in (ek, ev):
            if e.dtype != _BYTE or e.shape != want or not e.is_contiguous() or e.get_device() != dev:
                _refuse("exponents must be dense uint8 [pages, heads, page] on the cache's device")
        ek, ev = ek.data_ptr(), ev.data_ptr()
    l_shape, t_shape, s_shape = lengths.shape, table.shape, starts.shape
    if len(l_shape) != 1 or len(t_shape) != 2 or len(s_shape) != 1 or t_shape[0] != l_shape[0] or s_shape[0] != l_shape[0] + 1 or \
            starts.dtype != _INT or lengths.dtype != _INT or table.dtype != _INT:
        _refuse("table, starts and lengths must be int32 [batch, width], [batch + 1] and [batch]")
    batch, width = t_shape
    step, dense = table.stride()
    if (dense != 1 and width > 1) or not starts.is_contiguous() or not lengths.is_contiguous():
        _refuse("starts, lengths and the rows of the table must be dense")
    if starts.get_device() != dev or lengths.get_device() != dev or table.get_device() != dev:
        _refuse("table, starts and lengths must be on the cache's device")
    desc = capi.CacheDesc(pages, page, heads, d, code, batch, width, step, rows, k.data_ptr(), v.data_ptr(), ek, ev,
                          table.data_ptr(), starts.data_ptr(), lengths.data_ptr())
    return desc, code, dev, heads, d


def _packed(t, heads, d, dev, what):
    shape, s = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != heads or shape[2] != d or s[2] != 1 or t.get_device() != dev:
        _refuse(f"{what} must be [rows, {heads}, {d}] on the cache's device, the elements of a head neighbours")
    return capi.Packed(t.data_ptr(), s[0], s[1])


def cache_write(cache, k, v, table, starts, lengths, *, stream=None):
    """Writes the packed rows ``k`` and ``v`` [rows, heads, D] (float16 or bfloat16, each row and head on 16 bytes) to their positions.
    A 16-bit cache takes its own type.  A float8_e4m3fn cache is quantised as it is written: the scale of a token's head is the least
    power of two that brings its largest magnitude to 448 or less, codes are rounded to the nearest, ties to even; a row that holds an
    infinity or a NaN reads back as NaN.  A position must not be that of two rows (a page that two sequences name)."""
    if stream is None:
        r = calls.write(cache, k, v, table, starts, lengths)
        if r is not None:
            calls.result(r, k.get_device())
            return cache
    desc, code, dev, heads, d = _describe(cache, table, starts, lengths, k.shape[0])
    given = _codes().get(k.dtype)
    if given is None or given == capi.E4M3 or v.dtype != k.dtype or v.shape != k.shape or (code != capi.E4M3 and code != given):
        _refuse("keys and values must be float16 or bfloat16 rows of one shape, in the type of a 16-bit cache")
    pk, pv = _packed(k, heads, d, dev, "keys"), _packed(v, heads, d, dev, "values")
    context_for(dev).cache_write(desc, given, pk, pv, _stream_of(stream, dev))
    return cache


def cache_read(cache, table, starts, lengths, rows, *, dtype=None, out=None, stream=None):
    """The packed (keys, values) [rows, heads, D] at the positions of the packed rows, in ``dtype`` (float16 or bfloat16; a 16-bit cache
    gives its own).  ``lengths`` of zero read sequences from their first key on.  ``out``: a pair of tensors for them, columns of one buffer perhaps; in new ones, rows
    that belong to no sequence are undefined.  8-bit values beyond the type's range become its largest finite ones."""
    desc, code, dev, heads, d = _describe(cache, table, starts, lengths, rows)
    if dtype is None:
        dtype = out[0].dtype if out is not None else _torch().bfloat16 if code == capi.E4M3 else cache[0].dtype
    given = _codes().get(dtype)
    if given is None or given == capi.E4M3 or (code != capi.E4M3 and code != given):
        _refuse("rows are read as float16 or bfloat16, from a 16-bit cache in its own type")
    if out is None:
        like = cache[0]
        if stream is None:
            out = like.new_empty((2, rows, heads, d), dtype=dtype).unbind()
        else:
            with _on_stream(stream, like.device):
                out = like.new_empty((2, rows, heads, d), dtype=dtype).unbind()
    elif len(out) != 2 or any(t.dtype != dtype or t.shape[0] != rows for t in out):
        _refuse("out must be two tensors of the rows' type and count")
    pk, pv = _packed(out[0], heads, d, dev, "keys"), _packed(out[1], heads, d, dev, "values")
    context_for(dev).cache_read(desc, given, pk, pv, _stream_of(stream, dev))
    return tuple(out)


def cache_attention(cache, q, table, starts, lengths, *, mask=None, scale=None, max_new=0, tile_rows=0, out=None, stream=None):
    """Attention of the packed query rows ``q`` [rows, query heads, D] (float16 or bfloat16; a 16-bit cache has their type) over the
    cache, which holds their own keys and values already (``cache_write``).  A row sees the ``lengths[b]`` keys before the new tokens
    of its sequence and, of the new tokens, those up to itself, or those j for which ``mask[row, j]`` is set: ``mask`` is bool
    [rows, width], j counts within the sequence, and what lies beyond the width is not seen.  A single token is a tree of one.  Query
    head h reads key head h // (query heads / key heads).  A row that sees no key is zero; what a row does not see does not reach it,
    whatever it holds.  ``scale`` is 1 / sqrt(D) if not given.  ``max_new``, the largest number of new tokens of a sequence, helps the
    choice of a kernel, as the table's width does; ``tile_rows`` makes it: 16, 128 or 256 query rows (new tokens times query heads of a
    key head) a tile.  The kernels round weights differently, each to the 8 bits of bfloat16 or better (float16: 11).  ``out`` may be
    columns of the queries' buffer.  Rows of a new one that belong to no sequence are undefined."""
    shape = q.shape
    rows = shape[0]
    desc, code, dev, heads, d = _describe(cache, table, starts, lengths, rows)
    dtype = q.dtype
    given = _CODES.get(dtype)
    if given is None or given == capi.E4M3 or (code != capi.E4M3 and code != given):
        _refuse("queries must be float16 or bfloat16, in the type of a 16-bit cache")
    heads_q = shape[1] if len(shape) == 3 else 0
    if heads_q < 1 or heads_q % heads:
        _refuse("queries must be [rows, query heads, D], query heads a multiple of the key heads")
    width = step = 0
    mask_ptr = None
    if mask is not None:
        m_shape = mask.shape
        if mask.dtype != _torch().bool or len(m_shape) != 2 or m_shape[0] != rows or mask.get_device() != dev:
            _refuse("the mask must be bool [rows, width] on the cache's device")
        width = m_shape[1]
        step, dense = mask.stride()
        if dense != 1 and width > 1:
            _refuse("the rows of the mask must be dense")
        # (an empty tensor has no address; none of the new tokens is seen)
        mask_ptr = mask.data_ptr() if width else starts.data_ptr()
    pq = _packed(q, heads_q, d, dev, "queries")
    adesc = capi.CacheAttnDesc(heads_q, given, max_new, width, step, d ** -0.5 if scale is None else scale, tile_rows)
    if out is not None and (out.dtype != dtype or out.shape != shape):
        _refuse("out must have the type and shape of the queries")
    nbytes = capi.cache_attention_workspace_bytes(desc, adesc)
    if stream is None:
        if out is None:
            out = _new_like(q)
        workspace = _workspace(nbytes, dev)
    else:
        with _on_stream(stream, q.device):
            if out is None:
                out = _new_like(q)
            workspace = _workspace(nbytes, dev)
    po = _packed(out, heads_q, d, dev, "results")
    context_for(dev).cache_attention(desc, adesc, pq, po, mask_ptr, workspace.data_ptr(), nbytes, _stream_of(stream, dev))
    return out


def cache_check(device=None, *, stream=None):
    """Waits for the stream and raises RuntimeError where a kernel on it met a table entry out of range or gave up a wait."""
    torch = _torch()
    device = torch.device("cuda" if device is None else device)
    index = torch.cuda.current_device() if device.index is None else device.index
    with torch.cuda.device(index):
        context_for(index).check(_stream_ptr(stream, torch.device("cuda", index)))
