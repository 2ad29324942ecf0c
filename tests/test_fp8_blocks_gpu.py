"""The 8-bit block operators against their plain 64-bit forms: the block
quantizers bit for bit, the product, the fused SwiGLU and the norm step within
bounds counted in roundings, and a run of them together."""
import numpy as np
import pytest
import torch

import fp8_block_ref as ref
from fp8_block_ref import MAX, U32, U_BF16, block_absmax, dequant, nearest, spread, step, values

pytestmark = pytest.mark.gpu

F8 = {0: torch.float8_e4m3fn, 1: torch.float8_e5m2}
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _lib_ready(reng_lib):
    reng_lib.lib()


def randn(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def activations(seed, m, k, dtype=F32):
    x = randn(seed, m, k)
    x[:, ::97] *= 40.0
    return x.to(dtype)


def block_scale(top, fmt):
    """f32 scales: absmax / max_finite, no lower than the smallest normal f32, 1 for zeros."""
    s = (top / torch.tensor(MAX[fmt], device=top.device)).clamp(min=2.0 ** -126)
    return torch.where(top > 0, s, torch.ones_like(top))


def want_codes(x, rows, fmt):
    """Scales and values of encode(x / scale): the f32 quotient rounded to the format."""
    top = block_absmax(x.float(), rows)
    s = block_scale(top, fmt)
    q = x.float() / spread(s, rows, *x.shape)
    return nearest(q.double(), fmt), s


def pitched(rows, cols, pitch, dtype, offset=0, fill=None):
    """A [rows, cols] view of row pitch `pitch`, starting `offset` elements into its storage, and the storage."""
    t = torch.zeros(rows * pitch + offset + 64, device="cuda").to(dtype)
    if fill is not None:
        t.fill_(fill)
    return t[offset:offset + rows * pitch].view(rows, pitch)[:, :cols], t


# ------------------------------------------------------------- quantizers --
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (127, 72), (128, 128), (129, 1000), (300, 257),
                                       (37, 4096)])
def test_quantize_blocks_bit_for_bit(rows, cols, dtype, block_rows, fmt):
    from reng import fp8
    x = activations(rows + cols, rows, cols, dtype)
    codes, scales = fp8.quantize_blocks(x, block_rows, fmt)
    want, s = want_codes(x, block_rows, fmt)
    assert torch.equal(scales, s)
    got = values(fmt, "cuda")[codes.long()]
    assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("xoff,pitch,coff,cpitch", [(0, 160, 0, 152), (1, 131, 0, 160), (0, 136, 3, 131), (8, 144, 8, 136)])
def test_quantize_blocks_keeps_to_its_rows(block_rows, xoff, pitch, coff, cpitch):
    """Pitched and misaligned inputs and outputs; what lies between the rows is left as it was."""
    from reng import fp8
    rows, cols = 130, 130
    x, _ = pitched(rows, cols, pitch, BF16, xoff)
    x.copy_(activations(5, rows, cols, BF16))
    codes, store = pitched(rows, cols, cpitch, torch.uint8, coff, fill=0xA5)
    nb = -(-rows // block_rows)
    scales, sstore = pitched(nb, 2, 5, F32, 1, fill=7.5)
    fp8.quantize_blocks(x, block_rows, 0, codes=codes, scales=scales)
    want, s = want_codes(x.contiguous(), block_rows, 0)
    assert torch.equal(values(0, "cuda")[codes.long()], want) and torch.equal(scales, s)
    codes.fill_(0xA5)
    scales.fill_(7.5)
    assert bool((store == 0xA5).all()) and bool((sstore == 7.5).all())


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("fmt", [0, 1])
def test_quantize_blocks_special_values(block_rows, fmt):
    """Zeros, subnormals, infinities and NaN stay inside their own block."""
    from reng import fp8
    x = torch.zeros(128, 768, device="cuda")
    x[:, 128:256] = 1e-41 * randn(1, 128, 128)            # f32 subnormals
    x[:, 256:384] = randn(2, 128, 128)
    x[5, 300] = float("inf")
    x[:, 384:512] = randn(3, 128, 128)
    x[7, 400] = float("nan")
    x[:, 512:640] = 3e38 * torch.sign(randn(4, 128, 128))  # near the largest f32
    x[:, 640:] = randn(5, 128, 128)
    codes, scales = fp8.quantize_blocks(x, block_rows, fmt)
    got = values(fmt, "cuda")[codes.long()]
    top = block_absmax(x, block_rows)
    s = block_scale(top, fmt)
    assert torch.equal(scales, s)
    q = x / spread(s, block_rows, *x.shape)
    want = nearest(torch.nan_to_num(q.double(), nan=0.0), fmt)
    want[5, 300] = want[7, 400] = float("nan")  # inf / inf, and NaN itself
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want, nan=1e9))
    assert bool((got[:, :128] == 0).all())


# ---------------------------------------------------------------- product --
def operands(seed, m, n, k, xf=0, wf=0):
    from reng import fp8
    x, sx = fp8.quantize_blocks(activations(seed, m, k, BF16), 1, xf)
    w, sw = fp8.quantize_blocks(randn(seed + 1, n, k, scale=0.02, dtype=BF16), 128, wf)
    return x, sx, w, sw


def check_product(y, x, sx, w, sw, xf=0, wf=0):
    xd, wd = dequant(x, sx, 1, xf), dequant(w, sw, 128, wf)
    want = xd @ wd.T
    bound = ref.product_bound(xd, wd, sx.shape[1], y.dtype)
    err = (y.double() - want).abs()
    assert bool((err <= bound).all()), (float((err / bound.clamp(min=1e-300)).max()), float(err.max()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 64, 128), (1, 65, 127), (2, 127, 129), (7, 300, 1000),   # one tile, ragged everywhere
    (8, 128, 256), (9, 576, 1536), (33, 64, 512), (128, 64, 1024),          # K split over clusters
    (129, 200, 640), (1, 4096, 4096), (64, 1000, 2048), (100, 6144, 512),
    (300, 5120, 384), (1000, 2304, 256), (257, 40000, 136),                 # wider tiles
    (1024, 4096, 1024), (2050, 8200, 200),
])
def test_product(m, n, k, dtype):
    from reng import gemm
    ops = operands(m + n + k, m, n, k)
    check_product(gemm.gemm_fp8_blocks(*ops, dtype=dtype), *ops)


@pytest.mark.parametrize("m,n,k", [
    (1001, 5120, 384), (1001, 5123, 300), (2048, 6144, 128), (3000, 4100, 256), (5789, 909, 261),  # pairs
    (100, 40000, 200), (60, 40333, 128)])
def test_product_in_tiles_of_two_widths(m, n, k):
    """Sizes whose last round of tiles is narrower than the others."""
    from reng import gemm
    ops = operands(m + n + k, m, n, k)
    check_product(gemm.gemm_fp8_blocks(*ops, dtype=BF16), *ops)
    y, store = pitched(m, n, n + 3, F32, 1, fill=-3.0)  # by elements instead of whole boxes
    gemm.gemm_fp8_blocks(*ops, out=y)
    check_product(y, *ops)
    y.fill_(-3.0)
    assert bool((store == -3.0).all())


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("cols", [128, 131, 136])
def test_zeros_and_small_values_keep_their_sign(cols, fmt, block_rows):
    """-0 and negative values that round to zero take the code 0x80, positive ones 0, as the division gives them."""
    from reng import fp8
    for dtype in (BF16, F32):
        x = torch.zeros(128, cols, device="cuda", dtype=dtype)
        x[:, 1::2] = -0.0
        x[:, 0] = 3.0           # a scale
        x[:, 2], x[:, 3] = 1e-30, -1e-30
        codes, _ = fp8.quantize_blocks(x, block_rows, fmt)
        neg = torch.zeros_like(codes)
        neg[:, 1::2] = 0x80
        assert torch.equal(codes[:, 1:128], neg[:, 1:128]) and bool((codes[:, 128:] & 0x7F == 0).all())


@pytest.mark.parametrize("m,n,k", [(1, 6144, 512), (8, 5120, 777), (3, 4737, 384), (16, 4096, 640), (11, 2370, 200)])
def test_product_of_few_rows_in_small_ctas(m, n, k):
    """Widths between two sizes of a launch, which 4 warps a CTA hold at once."""
    from reng import gemm
    ops = operands(m + n + k, m, n, k)
    for dtype in (BF16, F32):
        check_product(gemm.gemm_fp8_blocks(*ops, dtype=dtype), *ops)


@pytest.mark.parametrize("xf,wf", [(0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("m,n,k", [(5, 200, 700), (300, 2000, 300), (1024, 6144, 256)])
def test_product_formats(m, n, k, xf, wf):
    from reng import gemm
    ops = operands(7, m, n, k, xf, wf)
    check_product(gemm.gemm_fp8_blocks(*ops, dtype=F32, x_fmt=xf, w_fmt=wf), *ops, xf, wf)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k", [(5, 100, 300), (200, 700, 260), (1024, 5000, 130)])
def test_product_pitches(m, n, k, dtype):
    """Operands inside larger matrices and a misaligned, pitched output whose surroundings stay as they were."""
    from reng import gemm
    x0, sx0, w0, sw0 = operands(11, m, n, k)
    pk = -(-k // 16) * 16 + 48
    x, xs = pitched(m, k, pk, torch.uint8, 16, fill=0x7F)   # NaN codes around the operands are never read
    w, ws = pitched(n, k, pk, torch.uint8, 32, fill=0x7F)
    x.copy_(x0), w.copy_(w0)
    sx, _ = pitched(m, sx0.shape[1], sx0.shape[1] + 3, F32, 1, fill=float("nan"))
    sw, _ = pitched(sw0.shape[0], sw0.shape[1], sw0.shape[1] + 1, F32, 3, fill=float("nan"))
    sx.copy_(sx0), sw.copy_(sw0)
    y, store = pitched(m, n, n + 5, dtype, 1, fill=-3.0)
    gemm.gemm_fp8_blocks(x, sx, w, sw, out=y)
    check_product(y, x0, sx0, w0, sw0)
    y.fill_(-3.0)
    assert bool((store == -3.0).all())


def test_product_is_deterministic_and_split_free_of_order():
    from reng import gemm
    ops = operands(3, 3, 576, 4096)
    a = gemm.gemm_fp8_blocks(*ops, dtype=F32)
    for _ in range(20):
        assert torch.equal(a, gemm.gemm_fp8_blocks(*ops, dtype=F32))


@pytest.mark.parametrize("m,n,k", [(4, 200, 512), (300, 4000, 256)])
def test_product_nan_stays_in_its_row(m, n, k):
    """A NaN code of x makes its own row NaN, one of w its own column, and nothing else."""
    from reng import gemm
    x, sx, w, sw = operands(13, m, n, k)
    x, w = x.clone(), w.clone()
    x[2, 130] = 0x7F
    w[77, 5] = 0x7F
    y = gemm.gemm_fp8_blocks(x, sx, w, sw, dtype=F32)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[2, :] = True
    bad[:, 77] = True
    assert torch.equal(torch.isnan(y), bad)


def test_product_of_no_rows():
    from reng import fp8, gemm
    w, sw = fp8.quantize_blocks(randn(1, 64, 256), 128)
    x = torch.empty((0, 256), dtype=torch.uint8, device="cuda")
    y = gemm.gemm_fp8_blocks(x, torch.empty((0, 2), device="cuda"), w, sw)
    assert y.shape == (0, 64)
    assert fp8.quantize_blocks(torch.empty((0, 256), device="cuda"))[0].shape == (0, 256)


# ----------------------------------------------------------------- SwiGLU --
SWIGLU_REL = 12 * U32


def check_groups(codes, scales, h, fmt, rel):
    """codes, scales of values known to `rel` relative: the scale to rel and a
    rounding, every code within half a step of its value over the scale given."""
    top = block_absmax(h, 1)
    s = torch.where(top > 0, top / MAX[fmt], torch.ones_like(top))
    assert bool(((scales.double() - s).abs() <= s * (rel + 2 * U32)).all())
    v = h / spread(scales.double(), 1, *h.shape)
    got = values(fmt, "cuda")[codes.long()]
    half = 0.5 * torch.maximum(step(v, fmt), step(got, fmt))
    assert bool(((got - v).abs() <= half + (rel + 2 * U32) * v.abs()).all())


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 14336), (5, 130), (33, 576), (700, 1536)])
def test_swiglu_quantize(rows, cols, dtype, fmt):
    from reng import fp8
    both = (4 * activations(rows, rows, 2 * cols)).to(dtype)
    both[0, 0] = -100.0  # exp(100) overflows f32: the product is zero there
    codes, scales = fp8.swiglu_quantize(both, fmt)
    g, u = both[:, :cols].double(), both[:, cols:].double()
    # 2^hi to 2^-22 (4 roundings), its correction, the sum and the two products one each,
    # the reciprocal to 2^-23 (2): at most SWIGLU_REL of 12 roundings
    h = g / (1 + torch.exp(-g)) * u
    h = torch.where(h.abs() < 1e-35, torch.zeros_like(h), h)
    check_groups(codes, scales, h, fmt, SWIGLU_REL)


# ------------------------------------------------------------------- norm --
# The mean square is a sum of non-negative terms: a thread adds at most 40 in
# sequence and the CTA 5 + 32 more, so it is 80 roundings off at most and its
# inverse root half of that; the division, the root, the gain, the gate and
# the products add at most 8.
NORM_REL = 48 * U32


def norm_case(rows, cols, btype, rtype, post, gate, seed=0):
    r = 3 * activations(seed, rows, cols)
    b = activations(seed + 1, rows, cols)
    g = {"none": None, "row": torch.rand(cols, device="cuda").to(btype),
         "full": torch.rand(rows, cols, device="cuda").to(rtype)}[gate]
    return dict(residual=r.to(rtype), branch=b.to(btype), gate=g,
                post_gain=1 + 0.1 * randn(seed + 2, cols) if post else None, pre_gain=1 + 0.1 * randn(seed + 3, cols))


def want_y(c, scale, eps):
    u = c["branch"].double()
    if c["post_gain"] is not None:
        u = u / (u.square().mean(1, keepdim=True) + eps).sqrt() * c["post_gain"].double()
    if c["gate"] is not None:
        u = u * c["gate"].double()
    return c["residual"].double() + scale * u, (scale * u).abs()


def want_h(y, gain, eps):
    h = y.double() / (y.double().square().mean(1, keepdim=True) + eps).sqrt()
    return h if gain is None else h * gain.double()


def check_y(y, c, scale, eps):
    want, mag = want_y(c, scale, eps)
    bound = NORM_REL * mag + 2 * U32 * want.abs()
    if y.dtype == BF16:
        bound = bound * (1 + U_BF16) + U_BF16 * want.abs()
    assert bool(((y.double() - want).abs() <= bound).all())


NORM_SHAPES = [(1, 1), (1, 128), (3, 129), (5, 4096), (33, 576), (2, 5120), (7, 8200), (2, 16384), (1, 32776), (130, 257)]


@pytest.mark.parametrize("post,gate", [(False, "none"), (True, "row"), (True, "full"), (False, "full")])
@pytest.mark.parametrize("btype,rtype,htype", [(BF16, BF16, BF16), (F32, BF16, F32), (F32, F32, BF16)])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_block_norm(rows, cols, btype, rtype, htype, post, gate):
    from reng import norm
    c = norm_case(rows, cols, btype, rtype, post, gate, rows + cols)
    y, h = norm.block_norm(**c, scale=0.22, eps=1e-6, dtype=htype)
    check_y(y, c, np.float32(0.22).item(), 1e-6)
    want = want_h(y, c["pre_gain"], 1e-6)
    bound = NORM_REL * want.abs() + (U_BF16 * (1 + NORM_REL) * want.abs() if htype == BF16 else 0)
    assert bool(((h.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("btype,rtype", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_block_norm_fp8(rows, cols, btype, rtype, fmt):
    from reng import norm
    c = norm_case(rows, cols, btype, rtype, True, "row", rows + cols)
    y, codes, scales = norm.block_norm_fp8(**c, scale=-1.5, eps=1e-5, fmt=fmt)
    check_y(y, c, -1.5, 1e-5)
    check_groups(codes, scales, want_h(y, c["pre_gain"], 1e-5), fmt, NORM_REL)


@pytest.mark.parametrize("cols", [576, 577, 40000])
def test_block_norm_in_place_and_without_parts(cols):
    from reng import norm
    c = norm_case(9, cols, BF16, BF16, True, "none", 3)
    y, h = norm.block_norm(**c)
    r = c["residual"].clone()
    y2, h2 = norm.block_norm(**{**c, "residual": r}, out=r)
    assert y2 is r and torch.equal(r, y) and torch.equal(h, h2)
    y3, none = norm.block_norm(**{**c, "pre_gain": None}, norm=False)
    assert none is None and torch.equal(y3, y)
    same, h3 = norm.block_norm(y, pre_gain=c["pre_gain"])
    assert same is y and torch.equal(h3, h)
    _, h4 = norm.block_norm(y)
    want = want_h(y, None, 1e-5)
    assert bool(((h4.double() - want).abs() <= (U_BF16 + NORM_REL * 2) * want.abs()).all())


def test_block_norm_pitches_leave_the_rest():
    from reng import norm
    rows, cols = 6, 264
    for off, pitch in ((0, 272), (1, 271)):
        c = norm_case(rows, cols, BF16, BF16, True, "full", 4)
        want = norm.block_norm(**c)
        moved = {}
        for k in ("residual", "branch", "gate"):
            moved[k], _ = pitched(rows, cols, pitch, BF16, off)
            moved[k].copy_(c[k])
        y, ys = pitched(rows, cols, pitch, BF16, off, fill=9.0)
        h, hs = pitched(rows, cols, pitch, BF16, off, fill=9.0)
        norm.block_norm(**{**c, **moved}, out=y, h=h)
        # another order of the sums may move y by one bf16 step, and h by that and a step of its own
        for got, w, steps in ((y, want[0], 1), (h, want[1], 2)):
            assert bool(((got.float() - w.float()).abs() <= steps * 2.02 * U_BF16 * w.float().abs() + 1e-30).all())
        y.fill_(9.0), h.fill_(9.0)
        assert bool((ys == 9.0).all()) and bool((hs == 9.0).all())


@pytest.mark.parametrize("rows,cols", [(8000, 75), (4000, 300), (1200, 1407), (700, 6200), (310, 8200)])
def test_block_norm_rows_of_any_alignment(rows, cols):
    """Several rows per team, each stream with a pitch and an offset of its own."""
    from reng import norm
    c = norm_case(rows, cols, F32, BF16, True, "full", cols)
    for i, k in enumerate(("residual", "branch", "gate")):
        moved, _ = pitched(rows, cols, cols + 3 + i, c[k].dtype, 1 + 2 * i, fill=float("nan"))
        moved.copy_(c[k])
        c[k] = moved
    for k in ("post_gain", "pre_gain"):
        moved = torch.empty(cols + 1, device="cuda")[1:]
        c[k] = moved.copy_(c[k])
    y, ys = pitched(rows, cols, cols + 2, BF16, 7, fill=9.0)
    h, hs = pitched(rows, cols, cols + 1, BF16, 2, fill=9.0)
    norm.block_norm(**c, scale=0.5, out=y, h=h)
    check_y(y, c, 0.5, 1e-5)
    want = want_h(y, c["pre_gain"], 1e-5)
    assert bool(((h.double() - want).abs() <= (NORM_REL + U_BF16 * (1 + NORM_REL)) * want.abs()).all())
    codes, cs = pitched(rows, cols, cols + 5, torch.uint8, 3, fill=0xA5)
    groups = (cols + 127) // 128
    scales, ss = pitched(rows, groups, groups + 1, F32, 1, fill=7.5)
    y2, _, _ = norm.block_norm_fp8(**c, scale=0.5, codes=codes, scales=scales)
    assert torch.equal(y2, y)
    check_groups(codes, scales, want_h(y2, c["pre_gain"], 1e-5), 0, NORM_REL)
    for t, store, fill in ((y, ys, 9.0), (h, hs, 9.0), (codes, cs, 0xA5), (scales, ss, 7.5)):
        t.fill_(fill)
        assert bool((store == fill).all())


@pytest.mark.parametrize("rows,cols", [(3000, 576), (3000, 577), (1001, 5120)])
def test_block_norm_in_place_over_many_rows(rows, cols):
    from reng import norm
    c = norm_case(rows, cols, BF16, BF16, True, "none", 5)
    y, h = norm.block_norm(**c)
    r = c["residual"].clone()
    y2, h2 = norm.block_norm(**{**c, "residual": r}, out=r)
    assert y2 is r and torch.equal(r, y) and torch.equal(h, h2)


def test_block_norm_rows_of_zeros():
    from reng import norm
    z = torch.zeros(4, 512, dtype=BF16, device="cuda")
    y, codes, scales = norm.block_norm_fp8(z, z, post_gain=torch.ones(512, device="cuda"))
    assert bool((y == 0).all()) and bool((codes == 0).all()) and bool((scales == 1).all())


# --------------------------------------------------------------- together --
def mlp(x_res, branch, wgu, wd, g, stream=None):
    """norm -> 8-bit gate/up -> SwiGLU -> 8-bit down, as a decoder's MLP runs them."""
    from reng import fp8, gemm, norm
    y, xc, xs = norm.block_norm_fp8(x_res, branch, pre_gain=g, stream=stream)
    gu = gemm.gemm_fp8_blocks(xc, xs, *wgu, stream=stream)
    hc, hs = fp8.swiglu_quantize(gu, stream=stream)
    return y, xc, xs, gu, hc, hs, gemm.gemm_fp8_blocks(hc, hs, *wd, dtype=F32, stream=stream)


def mlp_inputs(m, h=576, i=1536, seed=9):
    from reng import fp8
    return (activations(seed, m, h, BF16), activations(seed + 1, m, h, BF16),
            fp8.quantize_blocks(randn(seed + 2, 2 * i, h, scale=0.03, dtype=BF16), 128),
            fp8.quantize_blocks(randn(seed + 3, h, i, scale=0.03, dtype=BF16), 128), 1 + 0.1 * randn(seed + 4, h))


@pytest.mark.parametrize("m", [1, 8, 65, 700])
def test_a_run_of_them_together(m):
    """Each stage against its formula on the stage before's own output."""
    x, b, wgu, wd, g = mlp_inputs(m)
    y, xc, xs, gu, hc, hs, out = mlp(x, b, wgu, wd, g)
    check_groups(xc, xs, want_h(y, g, 1e-5), 0, NORM_REL)
    check_product(gu, xc, xs, *wgu)
    gate, up = gu[:, :1536].double(), gu[:, 1536:].double()
    check_groups(hc, hs, gate / (1 + torch.exp(-gate)) * up, 0, SWIGLU_REL)
    check_product(out, hc, hs, *wd)


@pytest.mark.parametrize("m", [1, 300])
def test_captured_replayed_and_on_another_stream(m):
    x, b, wgu, wd, g = mlp_inputs(m)
    want = [t.clone() for t in mlp(x, b, wgu, wd, g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mlp(x, b, wgu, wd, g)
    direct = mlp(x, b, wgu, wd, g, stream=side)
    side.synchronize()
    for a in (got, direct):
        assert all(torch.equal(p, q) for p, q in zip(want, a))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = mlp(x, b, wgu, wd, g)
        graphs.append((gr, out))
    x2 = activations(50, *x.shape, BF16)
    want2 = [t.clone() for t in mlp(x2, b, wgu, wd, g)]
    x.copy_(x2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):   # the two graphs at once: they share nothing
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(p, q) for p, q in zip(want2, out))


def test_products_of_every_kind_at_once():
    """Pairs of CTAs, K split over clusters, whole tiles and the few-row kernel
    on streams of their own, beside norms that fill shared memory."""
    from reng import gemm, norm
    sizes = [(1001, 5120, 1024), (64, 4096, 2048), (100, 6144, 512), (8, 2048, 4096), (300, 2000, 700)]
    sets = [operands(i, *mnk) for i, mnk in enumerate(sizes)]
    x = activations(3, 500, 4096, BF16)
    work = [lambda o=o: (gemm.gemm_fp8_blocks(*o, dtype=BF16),) for o in sets] + [lambda: norm.block_norm_fp8(x, x)]
    want = [w() for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[] for _ in work]
    for _ in range(10):
        for i, (w, st) in enumerate(zip(work, streams)):
            with torch.cuda.stream(st):
                got[i].append(w())
    torch.cuda.synchronize()
    for ref, runs in zip(want, got):
        assert all(torch.equal(a, b) for run in runs for a, b in zip(ref, run))


def test_offsets_past_32_bits():
    """Rows 2^30 and more elements apart."""
    from reng import fp8, gemm, norm
    pitch = (1 << 30) + 16
    x = activations(1, 5, 1000, BF16)
    far = torch.empty(4 * pitch + 1000, dtype=BF16, device="cuda").as_strided((5, 1000), (pitch, 1))
    far.copy_(x)
    for rows in (1, 128):
        for a, b in zip(fp8.quantize_blocks(far, rows), fp8.quantize_blocks(x, rows)):
            assert torch.equal(a, b)
    both = far[:, :512]
    for a, b in zip(fp8.swiglu_quantize(both), fp8.swiglu_quantize(x[:, :512].contiguous())):
        assert torch.equal(a, b)
    for n in (1000, 999):  # in pieces and by elements
        for a, b in zip(norm.block_norm(far[:, :n], x[:, :n], gate=far[:, :n]),
                        norm.block_norm(x[:, :n], x[:, :n], gate=x[:, :n])):
            assert torch.equal(a, b)
    del far, both
    for m in (5, 40):  # the few-row kernel and the tensor core's
        o = operands(2, m, 300, 256)
        p = (1 << 31) // (m - 1) // 16 * 16 + 4096
        c = torch.empty((m - 1) * p + 256, dtype=torch.uint8, device="cuda").as_strided((m, 256), (p, 1))
        c.copy_(o[0])
        y = torch.empty((m - 1) * p + 300, dtype=F32, device="cuda").as_strided((m, 300), (p, 1))
        gemm.gemm_fp8_blocks(c, *o[1:], out=y)
        assert torch.equal(y, gemm.gemm_fp8_blocks(*o, dtype=F32))
        del c, y


def test_python_refuses_wrong_device_matrices():
    from reng import fp8, gemm, norm
    x, sx, w, sw = operands(3, 4, 200, 256)
    b = torch.zeros(4, 256, dtype=BF16, device="cuda")
    bad = [
        lambda: gemm.gemm_fp8_blocks(x, sx, w[:, :128], sw), lambda: gemm.gemm_fp8_blocks(x, sx[:, :1], w, sw),
        lambda: gemm.gemm_fp8_blocks(x, sx, w, sw[:1]), lambda: gemm.gemm_fp8_blocks(x, sx.double(), w, sw),
        lambda: gemm.gemm_fp8_blocks(x.view(torch.int8), sx, w, sw), lambda: gemm.gemm_fp8_blocks(x, sx, w.t(), sw),
        lambda: gemm.gemm_fp8_blocks(x, sx, w, sw, dtype=torch.float16),
        lambda: gemm.gemm_fp8_blocks(x, sx, w, sw, out=b), lambda: gemm.gemm_fp8_blocks(x.cpu(), sx, w, sw),
        lambda: fp8.quantize_blocks(b, 64), lambda: fp8.quantize_blocks(b.half()), lambda: fp8.quantize_blocks(b.t()),
        lambda: fp8.quantize_blocks(b, codes=x[:2]), lambda: fp8.swiglu_quantize(b[:, :255]),
        lambda: fp8.quantize_blocks(b.expand(2, 4, 256)), lambda: fp8.quantize_blocks(b[:1].expand(4, 256)),
        lambda: norm.block_norm(b, b[:2]), lambda: norm.block_norm(b, b, post_gain=torch.ones(255, device="cuda")),
        lambda: norm.block_norm(b, b, gate=b[:, :255]), lambda: norm.block_norm(b, gate=b),
        lambda: norm.block_norm(b, b, pre_gain=torch.ones(256)), lambda: norm.block_norm(b, b.half()),
        lambda: norm.block_norm(b, b, out=b.float())]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("call %d was not refused" % i)


def test_no_wait_ran_out(reng_lib):
    reng_lib.call("reng_gemm_fp8_blocks_status")
