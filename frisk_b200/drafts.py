"""Verification of drafted tokens: ``draft_verify``."""
import contextlib

from . import calls, capi
from .cache import _on_stream, _stream_of
from .calls import context_for
from .execute import _torch


def _refuse(what):
    raise ValueError("frisk-b200-draft: " + what)


_KINDS = None
_NOTHING = contextlib.nullcontext()


def _list(t, n, kind, dev, what):
    shape = t.shape
    if t.dtype != kind or len(shape) != 1 or shape[0] != n or t.get_device() != dev or not t.is_contiguous():
        _refuse(f"{what} must be dense {str(kind)[6:]} [{n}] on the probabilities' device")
    return t.data_ptr()


def draft_verify(tokens, parents, starts, target, draft, accept, sample, *, max_new, stream=None):
    """Which drafted tokens stand, and the token behind them: (kept int32 [batch, max_new], counts int32 [batch], next [batch] in the
    tokens' type).

    Sequence b's rows ``starts[b]`` .. ``starts[b + 1] - 1`` are the nodes of a tree, as ``cache_attention`` scores them with a mask: node 0 the
    token sampled last, node i > 0 a drafted token behind node ``parents[row]`` < i (``parents`` None: behind node i - 1).  ``target`` [rows, vocabulary]
    holds the target's probabilities of the token behind each row, ``draft`` those that the children of each row were drawn from independently, or None
    where they were picked otherwise (looked up, or the most likely ones): float32, float16 or bfloat16, rows of any pitch.

    From node 0 on, the children of a node are tried in their order: a child stands if its random number ``accept[row]`` (float32, in [0, 1)) is
    below the target's probability of it over the draft's; otherwise the draft's distribution is taken off the target's for the next child.
    Where none is left, the next token is drawn with ``sample[b]`` from what is left: the first whose running sum passes it.  So tokens are
    distributed as the target's, whatever the draft.  Sums have 64 bits.  A distribution that is 1 at one token verifies greedily.

    ``kept[b, :counts[b]]`` are the nodes that stand, node 0 first, -1 behind them: what ``cache_keep`` takes.  A sequence without rows has count 0
    and next -1, as one with more than ``max_new`` (1 to 1024) rows or rows out of range, for which ``cache_check`` raises.  Probabilities that are NaN or
    negative count as 0."""
    global _KINDS
    if stream is None:
        r = calls.verify(tokens, parents, starts, target, draft, accept, sample, max_new)
        if r is not None:
            return calls.result(r, target.get_device())
    if _KINDS is None:
        torch = _torch()
        _KINDS = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}, torch.int32, torch.int64, torch.float32
    codes, i32, i64, f32 = _KINDS
    dtype, shape, dev = target.dtype, target.shape, target.get_device()
    code = codes.get(dtype)
    if code is None or len(shape) != 2:
        _refuse("target must be float32, float16 or bfloat16 [rows, vocabulary]")
    rows, vocab = shape
    step, dense = target.stride()
    if dense != 1 and vocab > 1:
        _refuse("the rows of target must be dense")
    if dev < 0:
        _refuse("tensors must be on one CUDA device (there is no CPU path)")
    p_draft, draft_step = None, 0
    if draft is not None:
        if draft.dtype != dtype or draft.shape != shape or draft.get_device() != dev:
            _refuse("draft must have the type, shape and device of target")
        draft_step, dense = draft.stride()
        if dense != 1 and vocab > 1:
            _refuse("the rows of draft must be dense")
        p_draft = draft.data_ptr()
    if starts.dim() != 1 or starts.shape[0] < 1:
        _refuse("starts must be int32 [batch + 1]")
    batch, kind = starts.shape[0] - 1, tokens.dtype
    if kind != i64 and kind != i32:
        _refuse("tokens must be int32 or int64")
    p_tokens = _list(tokens, rows, kind, dev, "tokens")
    p_parents = None if parents is None else _list(parents, rows, i32, dev, "parents")
    p_starts = _list(starts, batch + 1, i32, dev, "starts")
    p_accept, p_sample = _list(accept, rows, f32, dev, "accept"), _list(sample, batch, f32, dev, "sample")
    if not 1 <= max_new <= 1024:
        _refuse("max_new must be between 1 and 1024")
    with _NOTHING if stream is None else _on_stream(stream, target.device):
        kept, counts, token = starts.new_empty((batch, max_new)), starts.new_empty(batch), tokens.new_empty(batch)
    desc = capi.VerifyDesc(rows, step, draft_step, batch, max_new, vocab, code, kind == i64)
    context_for(dev).draft_verify(desc, p_tokens, p_parents, p_starts, target.data_ptr(), p_draft, p_accept, p_sample, kept.data_ptr(), counts.data_ptr(),
                                  token.data_ptr(), _stream_of(stream, dev))
    return kept, counts, token
