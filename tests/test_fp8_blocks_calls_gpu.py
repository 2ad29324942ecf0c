"""Calls of the 8-bit block operators at the ends of their ranges, and around
other streams (see test_fp8_blocks_gpu.py for their values)."""
import pytest
import torch

from fp8_block_ref import MAX, U32, step, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib_ready(reng_lib):
    reng_lib.lib()


# As test_fp8_blocks_gpu.py counts the near range, 12 roundings: the far one takes
# the exponential of a fraction (4), its correction (2) and two products (2).
SWIGLU_REL = 12 * U32


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("cols", [1, 8, 128, 130])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_swiglu_of_far_gates(dtype, cols, fmt):
    """Rows of one gate each, from -80 to -210, with up values that bring the product back into the f32 range."""
    from reng import fp8
    gate = torch.tensor([-80.0, -86.9, -87.0, -87.5, -88.0, -88.5, -89.0, -90.25, -95.0, -103.0, -110.5, -125.0, -150.0, -173.0,
                         -174.0, -180.0, -199.0, -201.0, -210.0])
    up = torch.tensor([1e-3, 1.0, 1e10, -3e20, 1e30, -3e38])
    g, u = (t.reshape(-1, 1).to(dtype).cuda() for t in torch.meshgrid(gate, up, indexing="ij"))
    both = torch.cat([g.expand(-1, cols), u.expand(-1, cols)], 1).contiguous()
    codes, scales = fp8.swiglu_quantize(both, fmt)
    g, u = g.double(), u.double()
    h = g / (1 + torch.exp(-g)) * u
    # in f32: below half its smallest step a zero (scale 1, code 0), and scales no lower than its smallest normal;
    # rows within a factor of 4 of that half step may go either way
    edge = 2.0 ** -150
    zero, alive = (h.abs() < edge / 4).flatten(), (h.abs() > edge * 4).flatten()
    assert int(zero.sum()) > 10 and int(alive.sum()) > 10
    got = values(fmt, "cuda")[codes.long()]
    assert bool((got[zero] == 0).all()) and bool((scales[zero] == 1).all())
    # a group of equal values: its scale is their size over max_finite, its codes max_finite with h's sign
    s = (h.abs() / MAX[fmt]).clamp(min=2.0 ** -126)
    tiny = 2.0 ** -149 / MAX[fmt]  # a subnormal h is off by half a step of 2^-149, and so its quotient
    assert bool(((scales.double() - s).abs() <= s * (SWIGLU_REL + 2 * U32) + tiny)[alive].all())
    v = (h / s).expand(-1, cols)
    bound = 0.5 * torch.maximum(step(v, fmt), step(got, fmt)) + (SWIGLU_REL + 2 * U32) * v.abs() + 2.0 ** -149 / s
    assert bool(((got - v).abs() <= bound)[alive].all())


def test_swiglu_of_a_gate_does_not_depend_on_its_neighbours():
    """Gates about the border of the far form, by themselves and between rows beyond it."""
    from reng import fp8
    gate = torch.linspace(-88, -85.5, 20000, device="cuda").reshape(-1, 1)
    both = torch.cat([gate, torch.full_like(gate, 1e38)], 1)
    rows = torch.cat([both, torch.tensor([[-150.0, 1.0]], device="cuda").expand(len(gate), 2)], 1).reshape(-1, 2)
    alone = torch.cat([fp8.swiglu_quantize(b)[1] for b in both.split(1)])
    assert torch.equal(fp8.swiglu_quantize(rows)[1][::2], alone)
    assert torch.equal(fp8.swiglu_quantize(both)[1], alone)


def test_swiglu_of_infinite_gates():
    from reng import fp8
    inf = float("inf")
    both = torch.tensor([[inf, 2.0], [-inf, 2.0], [-300.0, 5.0], [300.0, -5.0], [float("nan"), 1.0]], device="cuda")
    codes, scales = fp8.swiglu_quantize(both)
    assert scales[0, 0] == inf and int(codes[0, 0]) & 0x7F == 0x7F       # inf / inf
    assert int(codes[1, 0]) & 0x7F == 0x7F and scales[1, 0] == 1         # -inf / inf: NaN, never the absmax
    assert int(codes[2, 0]) == 0x80 and scales[2, 0] == 1                # the zero of the limit, with its sign
    assert values(0)[int(codes[3, 0])] == -240 and abs(float(scales[3, 0]) - 6.25) <= 6.25 * 2 * U32
    assert int(codes[4, 0]) & 0x7F == 0x7F and scales[4, 0] == 1


# ------------------------------------------------- a product that gave up --
def test_a_wait_that_ran_out_on_another_stream_is_told(reng_lib):
    """The status waits for work of every stream (torch's do not block the legacy one), tells once, and clears."""
    from reng import gemm
    gemm.gemm_fp8_blocks_status()
    side = torch.cuda.Stream()
    reng_lib.call("reng_gemm_fp8_blocks_wait_check", side.cuda_stream)  # 2 s, still running below
    with pytest.raises(reng_lib.RengError, match="gave up") as e:
        gemm.gemm_fp8_blocks_status()
    assert e.value.code == reng_lib.RENG_E_TIMEOUT and side.query()
    gemm.gemm_fp8_blocks_status()
    gemm.gemm_fp8_blocks_status(torch.cuda.current_device())


# ------------------------------------------------------------ side streams --
@pytest.mark.parametrize("what", ["quantize", "swiglu", "product", "norm", "norm_fp8"])
def test_a_side_stream_holds_its_inputs(what):
    """Inputs dropped right after a call on a busy stream, and their memory taken by others."""
    from reng import fp8, gemm, norm
    g = torch.Generator(device="cuda").manual_seed(3)

    def inputs():
        g.manual_seed(3)
        x = torch.randn(512, 4096, generator=g, device="cuda")
        if what == "product":
            return fp8.quantize_blocks(x) + fp8.quantize_blocks(torch.randn(512, 4096, generator=g, device="cuda"), 128)
        return (x, x + 1) if what.startswith("norm") else (x,)
    call = {"quantize": fp8.quantize_blocks, "swiglu": fp8.swiglu_quantize, "product": gemm.gemm_fp8_blocks,
            "norm": norm.block_norm, "norm_fp8": norm.block_norm_fp8}[what]

    def outputs(r):
        return [r] if torch.is_tensor(r) else [t for t in r if t is not None]
    want = [t.clone() for t in outputs(call(*inputs()))]
    side = torch.cuda.Stream()
    args = inputs()
    sizes = [(t.untyped_storage().nbytes(),) for t in args]
    keep = [torch.full(n, 7, dtype=torch.uint8, device="cuda") for n in sizes]  # the kernel that writes below is loaded
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(int(1e9))  # half a second
    got = outputs(call(*args, stream=side))
    assert not side.query()
    del args
    keep += [torch.full(n, 7, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(2)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # and on a raw handle, whose caller keeps the inputs
    args = inputs()
    side.wait_stream(torch.cuda.current_stream())
    got = outputs(call(*args, stream=side.cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


# ---------------------------------------------------------------- refusals --
def test_python_refuses_what_is_no_matrix(reng_lib):
    from reng import fp8, gemm, norm
    x, sx = fp8.quantize_blocks(torch.ones(4, 256, device="cuda"))
    w, sw = fp8.quantize_blocks(torch.ones(200, 256, device="cuda"), 128)
    b = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: gemm.gemm_fp8_blocks(x, sx, w[0, 0], sw), lambda: gemm.gemm_fp8_blocks(x, sx, w[0], sw),
                 lambda: gemm.gemm_fp8_blocks(x[0], sx, w, sw), lambda: norm.block_norm(b[0]), lambda: norm.block_norm_fp8(b[0]),
                 lambda: fp8.swiglu_quantize(b[0])):
        with pytest.raises(ValueError):
            call()
    # what only the library sees: sizes of zero, numbers that are no finite f32
    for call in (lambda: norm.block_norm(b, eps=-1.0), lambda: norm.block_norm(b, b, scale=float("inf")),
                 lambda: norm.block_norm(b, b, scale=1e39), lambda: norm.block_norm(b, b, eps=-1e300),
                 lambda: gemm.gemm_fp8_blocks(x, sx, w[:0], sw[:0]), lambda: fp8.quantize_blocks(b[:, :0])):
        with pytest.raises(reng_lib.RengError):
            call()


# -------------------------------------------------------------- long rows --
# A thread adds 16 squares in f32 (8 and 1 in sequence) and its tiles in 64 bits, the CTA 5 + 16 more:
# 32 roundings of the sum at most, 16 of its root, and 8 as in test_fp8_blocks_gpu.py: below its 48.
@pytest.mark.parametrize("cols", [40000, 1 << 20, (1 << 24) + 8, (1 << 24) + 3])
@pytest.mark.parametrize("post", [False, True])
def test_the_norm_of_a_long_row(cols, post):
    """Equal values, whose running sum in f32 would be off by one way of rounding, and normal ones."""
    from reng import norm
    from test_fp8_blocks_gpu import NORM_REL
    for x in (torch.full((2, cols), 1.1, device="cuda"), torch.randn(2, cols, device="cuda")):
        gain = torch.full((cols,), 0.75, device="cuda") if post else None
        y, h = norm.block_norm(torch.zeros_like(x), x, post_gain=gain, scale=1.0, eps=1e-5, dtype=torch.float32)

        def root(t):  # row by row: 64-bit copies of a whole matrix are large
            return torch.stack([(r.double().square().mean() + 1e-5).sqrt() for r in t])
        want = x.double()
        if post:
            want = want / root(x)[:, None] * 0.75
        assert bool(((y.double() - want).abs() <= NORM_REL * want.abs()).all())
        want = y.double() / root(y)[:, None]
        assert bool(((h.double() - want).abs() <= NORM_REL * want.abs()).all())


# ---------------------------------------------- outputs in a larger matrix --
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(130, 1, 1), (282, 2, 3), (1356, 14, 130), (202, 1396, 40), (1323, 38, 32), (605, 5157, 256),
                                   (300, 2047, 300), (257, 64, 128), (1001, 5123, 100), (40, 301, 200), (100, 40003, 64)])
def test_a_product_writes_its_own_columns_alone(m, n, k, dtype):
    """Rows on 16 bytes whose width is no multiple of 16 bytes, at every pitch to the next two: what lies
    behind a row stays."""
    from reng import gemm
    from test_fp8_blocks_gpu import check_product, operands, pitched
    ops = operands(m + n, m, n, k)
    want = None
    for pitch in range(n, n + 17):
        y, store = pitched(m, n, pitch, dtype, 16, fill=-3.0)
        gemm.gemm_fp8_blocks(*ops, out=y)
        if want is None:
            check_product(y, *ops)
            want = y.clone()
        assert torch.equal(y, want)
        y.fill_(-3.0)
        assert bool((store == -3.0).all()), pitch


# --------------------------------------------------------------- the engine --
@pytest.mark.parametrize("case,T", [("gqa", 2100), ("bias and qk_norm", 70), ("bias and qk_norm", 2100)])
def test_engine_past_2048_positions_and_with_biases_before_the_norm(reng_lib, case, T):
    """Decode attention's kernel for engines of 2048 positions and more, and q/k norms behind
    biases, in the block-scaled mode: one layer against its 64-bit attention."""
    import numpy as np
    from reng.model import Engine
    from reng.synth import prompt_ids
    from test_decode_gpu import small_cfg
    from test_fp8_blocks_engine_gpu import BLOCKS, attention_oracle, see_through
    both = case == "bias and qk_norm"
    cfg = small_cfg(bias=both, num_hidden_layers=1)
    w = see_through(cfg, 7)
    if both:
        rng = np.random.default_rng(3)
        for k in ("qn", "kn"):
            w["layers"][0][k] = rng.uniform(0.2, 0.6, cfg.head_dim()).astype(np.float32)
    ids = prompt_ids(T, cfg.vocab_size, seed=T)
    want, bound = attention_oracle(cfg, w, ids, both)
    e = Engine(cfg, w, batch=2, capacity=2304, fp8=BLOCKS)
    H = cfg.hidden_size

    def check(got, rows):
        got = torch.from_numpy(np.ascontiguousarray(got[..., :H])).to(want.device).double().reshape(-1, H)
        err = (got - want[rows]).abs()
        assert bool((err <= bound[rows]).all()), "%d values off, worst %.3g of the bound" % (
            int((err > bound[rows]).sum()), float((err / bound[rows]).max()))
    check(e.prefill(1, ids, all_logits=True)[2], slice(None))
    e.reset()
    e.prefill(0, ids[:T // 3])
    e.prefill(1, ids[:T - 1])
    logits, _ = e.step_logits(np.array([ids[T // 3], ids[T - 1]], np.uint32))
    check(logits[0], slice(T // 3, T // 3 + 1))
    check(logits[1], slice(T - 1, T))
    e.close()
