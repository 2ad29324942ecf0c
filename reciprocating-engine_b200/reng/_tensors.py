"""Checks and launch of the operators that take torch CUDA tensors in place
(fp8.quantize_blocks, fp8.swiglu_quantize, gemm.gemm_fp8_blocks, norm.*).

Misuse that is visible on the host raises ValueError before the call; what
the library refuses raises _lib.RengError.  Inference only: what they return
carries no gradient.
"""
import torch

from . import _lib

U8, F32 = (torch.uint8,), (torch.float32,)
TYPES = {torch.bfloat16: _lib.RENG_TYPE_BF16, torch.float32: _lib.RENG_TYPE_F32}
GROUP = 128  # columns (and, of a weight block, rows) that share one scale


def groups(n):
    return -(-n // GROUP)


def index(t):
    """The CUDA device index of a tensor."""
    i = t.get_device()
    if i < 0:
        raise ValueError("a tensor is on %s, not on a CUDA device" % t.device)
    return i


def matrix(t, name, dtypes, dev, rows=None, cols=None):
    """Row pitch of a 2-D tensor on device `dev` whose rows are contiguous."""
    s = t.shape
    if len(s) == 2 and t.dtype in dtypes and t.get_device() == dev and (rows is None or (s[0] == rows and s[1] == cols)):
        s0, s1 = t.stride()
        if s1 == 1 or s[1] == 1:
            if s0 >= s[1]:
                return s0
            if s[0] <= 1:
                return s[1]
    return _refuse(t, name, dtypes, dev, rows, cols)


def _refuse(t, name, dtypes, dev, rows, cols):
    if t.dim() != 2 or (rows is not None and tuple(t.shape) != (rows, cols)):
        raise ValueError("%s has shape %s%s" % (name, tuple(t.shape), "" if rows is None else ", not %s" % ((rows, cols),)))
    if t.dtype not in dtypes:
        raise ValueError("%s is %s" % (name, t.dtype))
    if t.get_device() != dev:
        raise ValueError("%s is on %s, not on CUDA device %d" % (name, t.device, dev))
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError("%s: the elements of a row must be contiguous" % name)
    raise ValueError("%s: rows overlap (stride %d for %d columns)" % (name, t.stride(0), t.shape[1]))


def vector(t, name, n, dev):
    """A contiguous f32 [n] on `dev`, or None."""
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != n or t.dtype != torch.float32 or t.get_device() != dev or not t.is_contiguous():
        raise ValueError("%s must be a contiguous float32 [%d] on CUDA device %d" % (name, n, dev))
    return t.data_ptr()


_empty = torch.empty


def codes_empty(rows, cols, device):
    """uint8 [rows, cols] in rows of 16-byte pitch (as the product reads them), and the pitch."""
    pitch = cols + 15 & -16
    if pitch == cols:
        return _empty(rows, cols, dtype=torch.uint8, device=device), cols
    return _empty(rows, pitch, dtype=torch.uint8, device=device)[:, :cols], pitch


try:  # the handle without building a Stream object around it, the device without an initialisation check
    from torch._C import _cuda_getCurrentRawStream as _raw_stream, _cuda_getDevice as _current
except ImportError:
    _current = torch.cuda.current_device

    def _raw_stream(dev):
        return torch.cuda.current_stream(dev).cuda_stream


def call(dev, name, *args):
    """The library call on the device's current stream, with the device current."""
    f = getattr(_lib.lib(), name)
    if dev == _current():
        rc = f(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = f(*args, _raw_stream(dev))
    if rc:
        _lib.check(rc)


def on_stream(stream, like, run, *args):
    """run(*args) on `stream` (a torch stream or a raw handle of the tensor's
    device): what it allocates belongs to that stream.  As with any work on a
    side stream, the caller orders it after its inputs.  The tensors among
    `args` are held until a torch stream is done with them; a raw handle may be
    gone by then, so its caller keeps them alive."""
    index(like)
    external = torch.cuda.ExternalStream
    if not isinstance(stream, torch.cuda.Stream):
        stream = external(stream, device=like.device)
    elif stream.device != like.device:
        raise ValueError("a stream of %s for tensors on %s" % (stream.device, like.device))
    with torch.cuda.stream(stream):
        out = run(*args)
    if not isinstance(stream, external):
        for t in args:
            if isinstance(t, torch.Tensor):
                t.record_stream(stream)
    return out


def blocks_out(x, dev, rows, cols, scale_rows, codes, scales):
    """Codes and scales of a block quantizer with their pitches, new where not given."""
    device = x.device
    if codes is None:
        codes, ldc = codes_empty(rows, cols, device)
    else:
        ldc = matrix(codes, "codes", U8, dev, rows, cols)
    if scales is None:
        lds = groups(cols)
        scales = _empty(scale_rows, lds, dtype=torch.float32, device=device)
    else:
        lds = matrix(scales, "scales", F32, dev, scale_rows, groups(cols))
    return codes, ldc, scales, lds


def quantize_blocks(x, block_rows, fmt, codes, scales):
    dev = index(x)
    ldx = matrix(x, "x", TYPES, dev)
    rows, cols = x.shape
    if block_rows == 1:
        sr = rows
    elif block_rows == GROUP:
        sr = groups(rows)
    else:
        raise ValueError("block_rows must be 1 or 128")
    codes, ldc, scales, lds = blocks_out(x, dev, rows, cols, sr, codes, scales)
    call(dev, "reng_fp8_quantize_blocks", x.data_ptr(), TYPES[x.dtype], rows, cols, ldx, block_rows, fmt,
         codes.data_ptr(), ldc, scales.data_ptr(), lds)
    return codes, scales


def swiglu_quantize(gate_up, fmt, codes, scales):
    dev = index(gate_up)
    ldx = matrix(gate_up, "gate_up", TYPES, dev)
    rows, both = gate_up.shape
    if both % 2:
        raise ValueError("gate_up has %d columns: not a gate and an up half" % both)
    cols = both // 2
    codes, ldc, scales, lds = blocks_out(gate_up, dev, rows, cols, rows, codes, scales)
    p = gate_up.data_ptr()
    call(dev, "reng_fp8_swiglu_quantize", p, p + cols * gate_up.element_size(), TYPES[gate_up.dtype], rows,
         cols, ldx, fmt, codes.data_ptr(), ldc, scales.data_ptr(), lds)
    return codes, scales


def gemm_fp8_blocks(x, x_scales, w, w_scales, out, dtype, x_fmt, w_fmt):
    dev = index(x)
    ldx = matrix(x, "x", U8, dev)
    M, K = x.shape
    N = w.shape[0] if w.dim() == 2 else _refuse(w, "w", U8, dev, None, None)
    kb = groups(K)
    ldw = matrix(w, "w", U8, dev, N, K)
    ldsx = matrix(x_scales, "x_scales", F32, dev, M, kb)
    ldsw = matrix(w_scales, "w_scales", F32, dev, groups(N), kb)
    if out is None:
        out = _empty(M, N, dtype=dtype or torch.bfloat16, device=x.device)
        ldy = N
    else:
        if dtype is not None and out.dtype != dtype:
            raise ValueError("out is %s, not %s" % (out.dtype, dtype))
        ldy = matrix(out, "out", TYPES, dev, M, N)
    if out.dtype not in TYPES:
        raise ValueError("out is %s" % out.dtype)
    call(dev, "reng_gemm_fp8_blocks", x.data_ptr(), ldx, x_scales.data_ptr(), ldsx, x_fmt, w.data_ptr(), ldw,
         w_scales.data_ptr(), ldsw, w_fmt, M, N, K, out.data_ptr(), TYPES[out.dtype], ldy)
    return out
