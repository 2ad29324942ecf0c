"""Plain 64-bit forms of the 8-bit block operators for their tests (torch, any
device): FP8 values from their bit fields, rounding by definition, block
scales, the product and the norm step, one formula at a time."""
import torch

GROUP = 128
MAX = {0: 240.0, 1: 57344.0}   # largest finite value of E4M3 (0) and E5M2 (1)
U32 = 2.0 ** -24               # half a step of f32, relative
U_BF16 = 2.0 ** -8


def pow2(e):
    """2^e exactly (a device's pow may be a step off), e an integer tensor within +-1000."""
    table = torch.tensor([2.0 ** i for i in range(-1000, 1001)], dtype=torch.float64, device=e.device)
    return table[e.long() + 1000]


def values(fmt, dev="cpu"):
    """f64 value of every code; the reserved top field of E5M2 as inf / NaN and
    E4M3's 0x7f / 0xff as NaN (0x78..0x7e read as 256..448, the tensor core's)."""
    mant, bias = (3, 7) if fmt == 0 else (2, 15)
    c = torch.arange(256, device=dev)
    f, m = (c & 127) >> mant, (c & ((1 << mant) - 1)).double() / (1 << mant)
    v = torch.where(f > 0, (1 + m) * pow2(f - bias), m * 2.0 ** (1.0 - bias))
    if fmt == 0:
        v[127] = v[255] = float("nan")
    else:
        v[[124, 252]] = float("inf")
        v[125:128] = v[253:256] = float("nan")
    return torch.where(c > 127, -v, v)


def step(v, fmt):
    """Spacing of the format's values at |v|."""
    mant, low = (3, -6) if fmt == 0 else (2, -14)
    e = torch.frexp(v)[1] - 1
    return pow2(e.clamp(min=low, max=900) - mant)


def nearest(v, fmt):
    """v (f64) to the nearest value, ties to even, saturating."""
    st = step(v, fmt)
    return (torch.round(v / st) * st).clamp(-MAX[fmt], MAX[fmt])


def spread(scales, rows, m, k):
    return scales.repeat_interleave(rows, 0)[:m].repeat_interleave(GROUP, 1)[:, :k]


def block_absmax(x, rows):
    m, k = x.shape
    pad = torch.nn.functional.pad(x, (0, -k % GROUP, 0, -m % rows))
    a = pad.reshape(pad.shape[0] // rows, rows, -1, GROUP).abs()
    return torch.nan_to_num(a, nan=0.0, posinf=float("inf")).amax((1, 3))


def dequant(codes, scales, rows, fmt):
    """f64 values of codes times their scales."""
    m, k = codes.shape
    return values(fmt, codes.device)[codes.long()] * spread(scales.double(), rows, m, k)


def product_bound(x, w, kb, out):
    """How far an output of the product may be off: each block's 128 exact
    products are summed in f32 (at most one rounding of up to a full step, 2
    U32, per term), its sum is scaled (one rounding of the scale, one of the
    FMA per block) and up to 8 partials are added."""
    mag = x.abs() @ w.abs().T
    b = (256 + kb + 10) * U32 * mag
    return b if out == torch.float32 else b * (1 + U_BF16) + U_BF16 * (x @ w.T).abs()
