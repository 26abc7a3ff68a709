"""Pages of a cache that sequences share: ``page_tables``, ``cache_fork``, ``cache_grow``, ``cache_keep``, ``cache_copy`` and ``cache_compact``.

``users`` (int32 [pages]) counts the table entries that name a page; 0 says that it is free.  A table entry below 0 names none.  A step of a
server is then

    users, table, lengths = cache_fork(cache, users, table, lengths, parents)         # beams change places, sequences end
    users, table, granted = cache_grow(cache, users, table, starts, lengths)          # room for the new tokens
    cache_write(cache, k, v, table, starts, lengths); cache_attention(cache, q, table, starts, lengths, mask=...)
    kept, counts, token = draft_verify(...)
    lengths = cache_keep(cache, table, starts, lengths, kept, counts)                 # the accepted ones move together

Tables live on the device and results follow from their contents alone, whatever the order of threads.  Results are new tensors; ``out``
takes tensors for them, which may be the inputs (in place), so that a captured step can be replayed.  The three results of one call may share an
allocation (with up to 64 KB of scratch), which lives as long as any of them: clone ``granted`` or ``lengths`` to keep it for longer than the table.  Contents are checked by the
kernels: what is out of range is left out, and ``cache_check`` raises.
"""
import contextlib

from . import calls, capi
from .cache import _codes, _on_stream, _refuse, _stream_of, _workspace
from .calls import context_for
from .execute import _torch

_NOTHING = contextlib.nullcontext()


def page_tables(cache, batch, width):
    """(users, table, lengths) of ``batch`` sequences without pages, ``width`` pages each at most, beside ``cache``: all pages are free."""
    torch = _torch()
    if batch < 0 or width < 0:
        _refuse("sizes outside the contract")
    made = dict(dtype=torch.int32, device=cache[0].device)
    return torch.zeros(cache[0].shape[0], **made), torch.full((batch, width), -1, **made), torch.zeros(batch, **made)


_INT = _BYTE = None


def _held(cache):
    """(element code, device index, [pages, heads, page, D], pointers of the four tensors), checked."""
    global _INT, _BYTE
    if _INT is None:
        _INT, _BYTE = _torch().int32, _torch().uint8
    parts = len(cache)
    if parts == 2:
        k, v = cache
        p_ek = p_ev = None
    elif parts == 4:
        k, v, ek, ev = cache
    else:
        _refuse("a cache is (k, v), or (k, v, k exponents, v exponents)")
    dtype, shape, dev = k.dtype, k.shape, k.get_device()
    code = _codes().get(dtype)
    if code is None or (code == capi.E4M3) != (parts == 4):
        _refuse("a cache holds float16, bfloat16, or float8_e4m3fn with exponents")
    if len(shape) != 4 or v.shape != shape or v.dtype != dtype or not k.is_contiguous() or not v.is_contiguous():
        _refuse("keys and values must be dense [pages, heads, page, D] of one type")
    if dev < 0 or v.get_device() != dev:
        _refuse("tensors must be on one CUDA device (there is no CPU path)")
    if parts == 4:
        want = shape[:3]
        for e in (ek, ev):
            if e.dtype != _BYTE or e.shape != want or not e.is_contiguous() or e.get_device() != dev:
                _refuse("exponents must be dense uint8 [pages, heads, page] on the cache's device")
        p_ek, p_ev = ek.data_ptr(), ev.data_ptr()
    return code, dev, shape, (k.data_ptr(), v.data_ptr(), p_ek, p_ev)


def _ints(t, n, dev, what):
    """The address of a dense int32 tensor [n]."""
    shape = t.shape
    if t.dtype != _INT or len(shape) != 1 or shape[0] != n or t.get_device() != dev or not t.is_contiguous():
        _refuse(f"{what} must be dense int32 [{n}] on the cache's device")
    return t.data_ptr()


def _rows(t, dev, what):
    """(address, rows, width, pitch) of an int32 table."""
    shape = t.shape
    if t.dtype != _INT or len(shape) != 2 or t.get_device() != dev:
        _refuse(f"{what} must be int32 [batch, width] on the cache's device")
    step, dense = t.stride()
    if dense != 1 and shape[1] > 1:
        _refuse(f"the rows of {what} must be dense")
    return t.data_ptr(), shape[0], shape[1], step


_EVERY_ROW = 2 ** 31 - 1  # (calls that see no packed rows, only their counts)


def _cache_desc(held, table, starts, lengths):
    code, _, (pages, heads, page, d), (k, v, ek, ev) = held
    ptr, batch, width, step = table
    return capi.CacheDesc(pages, page, heads, d, code, batch, width, step, _EVERY_ROW, k, v, ek, ev, ptr, starts, lengths)


def _change(which, cache, users, table, starts, lengths, parents, out, stream):
    """fork, grow and compact: new (users, table, third), or those in ``out``."""
    if out is None and stream is None:
        r = calls.change(which, cache, users, table, starts, lengths, parents)
        if r is not None:
            return calls.result(r, users.get_device())
    held = _held(cache)
    dev, pages = held[1], held[2][0]
    rows = _rows(table, dev, "the table")
    batch, width = rows[1], rows[2]
    p_users = _ints(users, pages, dev, "users")
    p_lengths = None if lengths is None else _ints(lengths, batch, dev, "lengths")
    p_starts = None if starts is None else _ints(starts, batch + 1, dev, "starts")
    p_parents = None if parents is None else _ints(parents, batch, dev, "parents")
    n_third = 1 if which == capi.PAGES_COMPACT else batch
    desc = _cache_desc(held, rows, p_starts, p_lengths)
    nbytes = capi.cache_pages_workspace_bytes(desc, which)
    workspace = None
    with _NOTHING if stream is None else _on_stream(stream, users.device):
        if nbytes:
            workspace = _workspace(nbytes, dev)
        if out is None:
            out = new_users, new_table, third = users.new_empty(pages), table.new_empty((batch, width)), users.new_empty(n_third)
            tables = capi.PageTables(p_users, new_users.data_ptr(), new_table.data_ptr(), third.data_ptr(), width)
        else:
            if not isinstance(out, (tuple, list)) or len(out) != 3:
                _refuse("out must be three tensors")
            to = _rows(out[1], dev, "the new table")
            if to[1] != batch or to[2] != width:
                _refuse("the new table must have the shape of the old one")
            tables = capi.PageTables(p_users, _ints(out[0], pages, dev, "the new users"), to[0], _ints(out[2], n_third, dev, "the third result"), to[3])
    context_for(dev).cache_pages(which, desc, tables, p_parents, None if workspace is None else workspace.data_ptr(), nbytes, _stream_of(stream, dev))
    return tuple(out)


def cache_fork(cache, users, table, lengths, parents, *, out=None, stream=None):
    """The new (users, table, lengths): row b of the table becomes what row ``parents[b]`` was, -1 leaves it without pages.  So one call forks
    (several rows of one parent), reorders beams, ends sequences (-1), and gives back what lies behind the last key of a row (its own
    number).  No page is copied: rows share them until ``cache_grow``."""
    return _change(capi.PAGES_FORK, cache, users, table, None, lengths, parents, out, stream)


def cache_grow(cache, users, table, starts, lengths, *, out=None, stream=None):
    """The new (users, table) with pages for ``starts[b + 1] - starts[b]`` more keys of each sequence, and how many of these were granted, int32
    [batch].  Pages are taken lowest first, by sequences in their order.  A page that is going to be written and that other rows have too
    is replaced by a copy; where several of the call's sequences have it, the last keeps it if no one else does.  A sequence gets all that
    it asks for or, from the first that lacks pages on, nothing (0; others than those that need no page).  Where ``users`` contradicts the pages that
    would be written, ``cache_check`` raises: a sequence that names a page without users gets nothing, and a page that more of the call's rows
    name than it has users is left to all of them."""
    return _change(capi.PAGES_GROW, cache, users, table, starts, lengths, None, out, stream)


def cache_compact(cache, users, table, *, out=None, stream=None):
    """Moves the used pages to the lowest indices, and returns the new (users, table) and their number, int32 [1]: from there on all pages are
    free.  The k-th used page behind them becomes the k-th free one among them; the others stay."""
    return _change(capi.PAGES_COMPACT, cache, users, table, None, None, None, out, stream)


def cache_copy(cache, source, target, *, into=None, stream=None):
    """Copies page ``source[i]`` of ``cache`` to page ``target[i]`` of ``into`` (the cache itself if not given, or another of the same type and
    page): both int32 [n] on the device.  A page must not be target twice nor, in one cache, source and target.  Returns ``into``."""
    if stream is None:
        r = calls.copy(cache, source, target, cache if into is None else into)
        if r is not None:
            calls.result(r, source.get_device())
            return cache if into is None else into
    held = _held(cache)
    other = held if into is None else _held(into)
    dev, shape = held[1], source.shape
    if len(shape) != 1 or other[1] != dev:
        _refuse("source and target must be lists of pages, and both caches on one device")
    n = shape[0]
    a, b = _ints(source, n, dev, "source"), _ints(target, n, dev, "target")
    no_table = (None, 0, 0, 0)
    context_for(dev).cache_copy(_cache_desc(held, no_table, None, None), _cache_desc(other, no_table, None, None), a, b, n, _stream_of(stream, dev))
    return cache if into is None else into


def cache_keep(cache, table, starts, lengths, kept, counts, *, out=None, stream=None):
    """The new lengths after ``counts[b]`` of the new tokens of each sequence were accepted: the key and value at position
    ``lengths[b] + kept[b, i]`` move to ``lengths[b] + i``.  ``kept`` int32 [batch, width] ascends within a sequence (``draft_verify`` gives
    both); what is behind the counts does not matter.  Pages stay where they are.  ``out`` may be ``lengths``."""
    if out is None and stream is None:
        r = calls.keep(cache, table, starts, lengths, kept, counts)
        if r is not None:
            return calls.result(r, lengths.get_device())
    held = _held(cache)
    dev = held[1]
    rows, path = _rows(table, dev, "the table"), _rows(kept, dev, "kept")
    batch = rows[1]
    if path[1] != batch:
        _refuse("kept must have a row for each sequence")
    p_starts, p_lengths, p_counts = _ints(starts, batch + 1, dev, "starts"), _ints(lengths, batch, dev, "lengths"), _ints(counts, batch, dev, "counts")
    if out is None:
        with _NOTHING if stream is None else _on_stream(stream, lengths.device):
            out = lengths.new_empty(batch)
    p_out = _ints(out, batch, dev, "the new lengths")
    context_for(dev).cache_keep(_cache_desc(held, rows, p_starts, p_lengths), path[0], path[3], path[2], p_counts, p_out, _stream_of(stream, dev))
    return out
