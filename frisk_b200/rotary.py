"""Rotary positions of queries and keys: ``rotary``, its gradients ``rotary_backward``, and ``rotary_frequencies``.

Packed rows [tokens, heads, D], as a projection leaves them: queries and keys may be columns of one buffer, or lie side by side in each
head.  The first ``2 * len(frequencies)`` elements of every head are rotated in pairs, the others pass:

    (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t),    t = position * frequency
"""
import math

from . import capi
from .cache import _new_like, _on_stream, _stream_of
from .execute import _torch, context_for

_CODE = None


def rotary_frequencies(dim, base=10000.0, *, scaling=None, factor=1.0, trained=None, low=1.0, high=None, device="cuda"):
    """(frequencies, amplitude) for ``rotary``: radians per position of the ``dim // 2`` pairs, base ** (-2 i / dim), as a
    float64 tensor, and the factor on the rotated values.

    ``scaling`` stretches them to contexts ``factor`` times as long as the ``trained`` ones:

    * ``"linear"``      every pair turns ``factor`` times slower
    * ``"ntk"``         a larger base, with which the slowest pair turns ``factor`` times slower and the fastest stays
    * ``"wavelength"``  pairs with more than ``high`` (4) turns in the trained context stay, those with fewer than ``low`` turn
      ``factor`` times slower, the others in between by their number of turns
    * ``"yarn"``        the same with ``high`` 32, and amplitude 0.1 ln(factor) + 1.  (As the method was published; a model whose
      frequencies go over by the index of the pair instead needs its own, which ``rotary`` takes as well.)
    """
    if dim < 2 or dim % 2:
        raise ValueError("frisk-b200-rotary: dim must be even and positive")
    if scaling not in (None, "linear", "ntk", "wavelength", "yarn"):
        raise ValueError(f"frisk-b200-rotary: unknown scaling {scaling!r}")
    if not (base > 0 and factor >= 1.0):
        raise ValueError("frisk-b200-rotary: base must be positive and factor at least 1")
    if scaling == "ntk" and dim > 2:
        base *= factor ** (dim / (dim - 2))
    freq = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear" or (scaling == "ntk" and dim == 2):
        freq = [f / factor for f in freq]
    elif scaling in ("wavelength", "yarn"):
        if trained is None or trained <= 0:
            raise ValueError(f"frisk-b200-rotary: scaling {scaling!r} needs the trained context length")
        if high is None:
            high = 32.0 if scaling == "yarn" else 4.0
        if not high > low:
            raise ValueError("frisk-b200-rotary: high must be above low")
        stay = [min(1.0, max(0.0, (trained * f / (2 * math.pi) - low) / (high - low))) for f in freq]
        freq = [f * (s + (1.0 - s) / factor) for f, s in zip(freq, stay)]
    amplitude = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0
    return _torch().tensor(freq, dtype=_torch().float64, device=device), amplitude


def _refuse(what):
    raise ValueError("frisk-b200-rotary: " + what)


def _operand(t, dev, d):
    s = t.stride()
    if (s[2] != 1 and d > 1) or t.get_device() != dev:
        _refuse("operands must be on one device, the elements of a head neighbours")
    return capi.Packed(t.data_ptr(), s[0], s[1])


def _rotate(q, k, positions, frequencies, amplitude, interleaved, out, stream, inverse):
    global _CODE
    if _CODE is None:
        torch = _torch()
        _CODE = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}, torch.int64, torch.int32, torch.float64
    codes, i64, i32, f64 = _CODE
    dtype, shape, dev = q.dtype, q.shape, q.get_device()
    code = codes.get(dtype)
    if code is None:
        _refuse("elements must be float32, float16 or bfloat16")
    if len(shape) != 3:
        _refuse("queries and keys must be [tokens, heads, D]")
    n, heads_q, d = shape
    heads_k = 0
    if k is not None:
        k_shape = k.shape
        if k.dtype != dtype or len(k_shape) != 3 or k_shape[0] != n or k_shape[2] != d:
            _refuse("keys must have the queries' type, tokens and D")
        heads_k = k_shape[1]
    if out is None:
        if stream is None:
            q_out, k_out = _new_like(q), None if k is None else _new_like(k)
        else:
            with _on_stream(stream, q.device):
                q_out, k_out = _new_like(q), None if k is None else _new_like(k)
    else:
        if not isinstance(out, (tuple, list)) or len(out) != 2 or out[0] is None or (k is None) != (out[1] is None):
            _refuse("out must be a pair (None for absent keys)")
        q_out, k_out = out
        if q_out.dtype != dtype or q_out.shape != shape or (k is not None and (k_out.dtype != dtype or k_out.shape != k_shape)):
            _refuse("results must have the type and shape of what is rotated")
    p_type, p_shape, f_shape = positions.dtype, positions.shape, frequencies.shape
    if (p_type != i64 and p_type != i32) or len(p_shape) != 1 or p_shape[0] != n or not positions.is_contiguous():
        _refuse("positions must be int32 or int64, one for every token")
    if frequencies.dtype != f64 or len(f_shape) != 1 or not frequencies.is_contiguous():
        _refuse("frequencies must be one float64 for every pair")
    if dev < 0 or positions.get_device() != dev or frequencies.get_device() != dev:
        _refuse("operands must be on one CUDA device (there is no CPU path)")
    if n == 0:
        return q_out, k_out
    desc = capi.RotaryDesc(n, heads_q, heads_k, d, 2 * f_shape[0], code, interleaved, inverse, p_type == i64, amplitude)
    absent = heads_k == 0
    context_for(dev).rotary(desc, positions.data_ptr(), frequencies.data_ptr(), _operand(q, dev, d), None if absent else _operand(k, dev, d),
                            _operand(q_out, dev, d), None if absent else _operand(k_out, dev, d), _stream_of(stream, dev))
    return q_out, k_out


def rotary(q, k, positions, frequencies, *, amplitude=1.0, interleaved=False, out=None, stream=None):
    """The rotated (queries, keys).  ``q`` [tokens, heads, D] and ``k`` [tokens, key heads, D] (or None) in float32, float16 or
    bfloat16 with any strides of tokens and heads; ``positions`` int32 or int64 [tokens]; ``frequencies`` float64 [pairs].  Pairs are
    (i, i + pairs), or (2 i, 2 i + 1) if ``interleaved``.  Angles are reduced to one turn in 64 bits.  ``out`` is a pair of tensors
    for the results; one may be its input (in place)."""
    return _rotate(q, k, positions, frequencies, amplitude, interleaved, out, stream, False)


def rotary_backward(dq, dk, positions, frequencies, *, amplitude=1.0, interleaved=False, out=None, stream=None):
    """The gradients of ``rotary``'s inputs from those of its results: the transposed rotation, the same arguments.  (Neither is bound to
    autograd: results of ``rotary`` carry no history.)"""
    return _rotate(dq, dk, positions, frequencies, amplitude, interleaved, out, stream, True)
