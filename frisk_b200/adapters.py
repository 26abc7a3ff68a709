"""Low-rank adapters of many requests, added to a shared projection: ``adapter_gemm``."""
import contextlib

from . import calls, capi
from .cache import _new_like, _on_stream, _stream_of, _workspace
from .calls import context_for
from .execute import _torch

_KINDS = None
_NOTHING = contextlib.nullcontext()


def _refuse(what):
    raise ValueError("frisk-b200-adapter: " + what)


def adapter_gemm(x, a, b, c, starts, adapters, *, scales=None, out=None, stream=None):
    """``c[r] + scales[w] * (x[r] @ a[w].T) @ b[w].T`` for the packed rows r of sequence s, ``w = adapters[s]``; a sequence whose adapter is below 0
    has none.  Rows ``starts[s]`` .. ``starts[s + 1] - 1`` belong to sequence s; rows of no sequence are left as they are (undefined in a new tensor).

    ``x`` [rows, K], ``a`` [count, rank, K] and ``b`` [count, N, rank] are float16 or bfloat16, their rows on 16 bytes and the rank a multiple of 8 up to
    128 (pad it with zeros).  ``c`` [rows, N], the result of the shared projection (``gemm``), has their type or float32 and any pitch, and the result
    its type; ``out`` may be ``c``.  ``starts`` int32 [batch + 1], ``adapters`` int32 [batch] and ``scales`` float32 [count] (1 if not given) are on the device, so that a
    captured step can be replayed for other requests; an adapter out of range counts as none, and ``cache_check`` raises.  Sums have 32
    bits, those between the two products too, and the result is rounded once."""
    global _KINDS
    if out is None and stream is None:
        r = calls.adapters(x, a, b, c, starts, adapters, scales)
        if r is not None:
            return calls.result(r, x.get_device())
    if _KINDS is None:
        torch = _torch()
        _KINDS = {torch.float16: capi.F16, torch.bfloat16: capi.BF16}, torch.float32, torch.int32
    codes, f32, i32 = _KINDS
    dtype, to, dev = x.dtype, c.dtype, x.get_device()
    code = codes.get(dtype)
    if code is None or a.dtype != dtype or b.dtype != dtype:
        _refuse("x, a and b must be float16 or bfloat16")
    if to != dtype and to != f32:
        _refuse("c must have the type of x, or float32")
    sx, sa, sb, sc, batch = x.shape, a.shape, b.shape, c.shape, adapters.shape
    if len(sx) != 2 or len(sa) != 3 or len(sb) != 3 or len(sc) != 2:
        _refuse("x and c must be [rows, width], a [count, rank, K], b [count, N, rank]")
    rows, k = sx
    count, rank, _ = sa
    n = sb[1]
    if sa[2] != k or sb[0] != count or sb[2] != rank or sc[0] != rows or sc[1] != n:
        _refuse("x [rows, K], a [count, rank, K], b [count, N, rank] and c [rows, N] do not fit together")
    (ldx, x1), (a_step, lda, a1), (b_step, ldb, b1), (ldc, c1) = x.stride(), a.stride(), b.stride(), c.stride()
    if (k > 1 and (x1 != 1 or a1 != 1)) or b1 != 1 or (n > 1 and c1 != 1):
        _refuse("rows must be dense")
    if dev < 0 or a.get_device() != dev or b.get_device() != dev or c.get_device() != dev or starts.get_device() != dev or adapters.get_device() != dev:
        _refuse("tensors must be on one CUDA device (there is no CPU path)")
    if len(batch) != 1 or starts.shape != (batch[0] + 1,) or starts.dtype != i32 or adapters.dtype != i32 or not starts.is_contiguous() or not adapters.is_contiguous():
        _refuse("starts and adapters must be dense int32 [batch + 1] and [batch]")
    p_scales = None
    if scales is not None:
        if scales.dtype != f32 or scales.shape != (count,) or not scales.is_contiguous() or scales.get_device() != dev:
            _refuse("scales must be dense float32, one for each adapter, on the same device")
        p_scales = scales.data_ptr()
    ldo, workspace = n, None
    if out is not None:
        if out.dtype != to or out.shape != sc or out.get_device() != dev:
            _refuse("out must have the type, shape and device of c")
        ldo, dense = out.stride()
        if n > 1 and dense != 1:
            _refuse("rows must be dense")
    desc = capi.AdapterDesc(rows, k, n, ldx, lda, a_step, ldb, b_step, ldc, ldo, rank, count, batch[0], code, code if to == dtype else capi.F32)
    nbytes = capi.adapter_workspace_bytes(desc)
    with _NOTHING if stream is None else _on_stream(stream, c.device):
        if out is None:
            out = _new_like(c)
        if nbytes:
            workspace = _workspace(nbytes, dev)
    context_for(dev).adapter_gemm(desc, x.data_ptr(), a.data_ptr(), b.data_ptr(), c.data_ptr(), p_scales, starts.data_ptr(), adapters.data_ptr(), out.data_ptr(),
                                  None if workspace is None else workspace.data_ptr(), nbytes, _stream_of(stream, dev))
    return out
