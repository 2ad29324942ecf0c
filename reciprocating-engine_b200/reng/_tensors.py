"""Checks and launch of the operators that take torch CUDA tensors in place
(fp8.quantize_blocks, fp8.swiglu_quantize, gemm.gemm_fp8_blocks, norm.*).

Misuse that is visible on the host raises ValueError before the call; what
the library refuses raises _lib.RengError.
"""
import torch

from . import _lib

TYPES = {torch.bfloat16: _lib.RENG_TYPE_BF16, torch.float32: _lib.RENG_TYPE_F32}
GROUP = 128  # columns (and, of a weight block, rows) that share one scale


def groups(n):
    return -(-n // GROUP)


def matrix(t, name, dtypes, dev, shape=None):
    """Row pitch of a 2-D tensor on `dev` whose rows are contiguous."""
    if t.dim() != 2 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError("%s has shape %s%s" % (name, tuple(t.shape), "" if shape is None else ", not %s" % (shape,)))
    if t.dtype not in dtypes:
        raise ValueError("%s is %s" % (name, t.dtype))
    if t.device != dev or dev.type != "cuda":
        raise ValueError("%s is on %s, not on %s" % (name, t.device, dev if dev.type == "cuda" else "a CUDA device"))
    rows, cols = t.shape
    s0, s1 = t.stride()
    if s1 != 1 and cols > 1:
        raise ValueError("%s: the elements of a row must be contiguous" % name)
    if rows <= 1:
        return s0 if s0 >= cols else cols
    if s0 < cols:
        raise ValueError("%s: rows overlap (stride %d for %d columns)" % (name, s0, cols))
    return s0


def vector(t, name, n, dev):
    """A contiguous f32 [n] on `dev`, or None."""
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != n or t.dtype != torch.float32 or t.device != dev or not t.is_contiguous():
        raise ValueError("%s must be a contiguous float32 [%d] on %s" % (name, n, dev))
    return t.data_ptr()


def codes_empty(rows, cols, dev):
    """uint8 [rows, cols] in rows of 16-byte pitch, as the product reads them."""
    pitch = -(-cols // 16) * 16
    t = torch.empty((rows, pitch), dtype=torch.uint8, device=dev)
    return t if pitch == cols else t[:, :cols]


def call(dev, stream, name, *args):
    """The library call on `stream` (default: the device's current stream),
    with the tensors' device current."""
    st = torch.cuda.current_stream(dev).cuda_stream if stream is None else getattr(stream, "cuda_stream", stream)
    if dev.index == torch.cuda.current_device():
        _lib.call(name, *args, st)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, st)
