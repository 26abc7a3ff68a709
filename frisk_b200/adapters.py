"""Low-rank adapters of many requests, added to a shared projection: ``adapter_gemm``."""
import contextlib

from . import capi
from .cache import _new_like, _on_stream, _stream_of, _workspace
from .execute import _torch, context_for


def _refuse(what):
    raise ValueError("frisk-b200-adapter: " + what)


def adapter_gemm(x, a, b, c, starts, adapters, *, scales=None, out=None, stream=None):
    """``c[r] + scales[w] * (x[r] @ a[w].T) @ b[w].T`` for the packed rows r of sequence s, ``w = adapters[s]``; a sequence whose adapter is below 0
    has none.  Rows ``starts[s]`` .. ``starts[s + 1] - 1`` belong to sequence s; rows of no sequence are left as they are (undefined in a new tensor).

    ``x`` [rows, K], ``a`` [count, rank, K] and ``b`` [count, N, rank] are float16 or bfloat16, their rows on 16 bytes and the rank a multiple of 8 up to
    128 (pad it with zeros).  ``c`` [rows, N], the result of the shared projection (``gemm``), has their type or float32 and any pitch, and the result
    its type; ``out`` may be ``c``.  ``starts`` int32 [batch + 1], ``adapters`` int32 [batch] and ``scales`` float32 [count] (1 if not given) are on the device, so that a
    captured step can be replayed for other requests; an adapter out of range counts as none, and ``cache_check`` raises.  Sums have 32
    bits, and the result is rounded once."""
    torch = _torch()
    code = {torch.float16: capi.F16, torch.bfloat16: capi.BF16}.get(x.dtype)
    dev = x.get_device()
    if code is None or a.dtype != x.dtype or b.dtype != x.dtype:
        _refuse("x, a and b must be float16 or bfloat16")
    if c.dtype != x.dtype and c.dtype != torch.float32:
        _refuse("c must have the type of x, or float32")
    if x.dim() != 2 or a.dim() != 3 or b.dim() != 3 or c.dim() != 2:
        _refuse("x and c must be [rows, width], a [count, rank, K], b [count, N, rank]")
    (rows, k), (count, rank, _), n = x.shape, a.shape, b.shape[1]
    if a.shape[2] != k or b.shape[0] != count or b.shape[2] != rank or c.shape != (rows, n):
        _refuse("x [rows, K], a [count, rank, K], b [count, N, rank] and c [rows, N] do not fit together")
    if (k > 1 and (x.stride(1) != 1 or a.stride(2) != 1)) or b.stride(2) != 1 or (n > 1 and c.stride(1) != 1):
        _refuse("rows must be dense")
    if dev < 0 or any(t.get_device() != dev for t in (a, b, c, starts, adapters)) or (scales is not None and scales.get_device() != dev):
        _refuse("tensors must be on one CUDA device (there is no CPU path)")
    batch = adapters.shape[0] if adapters.dim() == 1 else -1
    if batch < 0 or starts.shape != (batch + 1,) or starts.dtype != torch.int32 or adapters.dtype != torch.int32 or not starts.is_contiguous() or \
            not adapters.is_contiguous():
        _refuse("starts and adapters must be dense int32 [batch + 1] and [batch]")
    if scales is not None and (scales.dtype != torch.float32 or scales.shape != (count,) or not scales.is_contiguous()):
        _refuse("scales must be dense float32, one for each adapter")
    if out is not None and (out.dtype != c.dtype or out.shape != c.shape or out.get_device() != dev or (n > 1 and out.stride(1) != 1)):
        _refuse("out must have the type, shape and device of c, and dense rows")
    with contextlib.nullcontext() if stream is None else _on_stream(stream, c.device):
        if out is None:
            out = _new_like(c)
        desc = capi.AdapterDesc(rows, k, n, x.stride(0), a.stride(1), a.stride(0), b.stride(1), b.stride(0), c.stride(0), out.stride(0), rank, count, batch, code,
                                code if c.dtype == x.dtype else capi.F32)
        nbytes = capi.adapter_workspace_bytes(desc)
        workspace = _workspace(nbytes, dev) if nbytes else None
    context_for(dev).adapter_gemm(desc, x.data_ptr(), a.data_ptr(), b.data_ptr(), c.data_ptr(), None if scales is None else scales.data_ptr(), starts.data_ptr(),
                                  adapters.data_ptr(), out.data_ptr(), None if workspace is None else workspace.data_ptr(), nbytes, _stream_of(stream, dev))
    return out
