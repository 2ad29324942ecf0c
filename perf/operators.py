"""What is measured of the 8-bit block operators: the quantizers, the block-scaled product and the
norm between two blocks, at the widths of the models this repository serves.

Each case names one operator (`op`) and its sizes.  `run` computes it in plain torch operations in
32 bits, or, with `own` set, through the framework's own calls.
"""
import math
import os
import sys

import torch

own = False

GROUP = 128                     # values (or rows and columns of a weight block) that share one scale
E4M3_MAX, E5M2_MAX = 240.0, 57344.0   # largest finite values of the framework's two formats
EPS = 1e-5

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "reciprocating-engine_b200")


def listed():
    return [
        # one token of a small model (SmolLM2-135M down_proj widths) for 13 sequences: latency alone counts
        {"name": "product_small", "op": "product", "m": 13, "n": 576, "k": 1536, "out": "f32", "xf": "e4m3", "wf": "e4m3"},
        # one sequence's next token through Llama-8B's q/k/v projection: the weights' bytes count
        {"name": "product_token", "op": "product", "m": 1, "n": 6144, "k": 4096, "out": "bf16", "xf": "e4m3", "wf": "e4m3"},
        # a decode step of 64 sequences through Llama-8B's gate and up projections
        {"name": "product_batch", "op": "product", "m": 64, "n": 28672, "k": 4096, "out": "bf16", "xf": "e4m3", "wf": "e4m3"},
        # the ragged last block of a prompt through Qwen2.5-32B's down projection
        {"name": "product_ragged", "op": "product", "m": 1001, "n": 5120, "k": 27648, "out": "f32", "xf": "e5m2", "wf": "e4m3"},
        # a long prompt through Llama-8B's gate and up projections: the tensor cores' rate counts
        {"name": "product_prompt", "op": "product", "m": 8192, "n": 28672, "k": 4096, "out": "bf16", "xf": "e4m3", "wf": "e4m3"},
        # between two blocks of one token: residual add, norm, 8-bit groups for the next product
        {"name": "norm_token", "op": "norm", "m": 1, "h": 4096, "branch": "bf16", "post": False, "gate": "none", "out": "e4m3"},
        # a ragged block of rows with norms on both sides, a gate per element and a residual scale
        {"name": "norm_both", "op": "norm", "m": 1023, "h": 5120, "branch": "f32", "post": True, "gate": "full", "out": "bf16"},
        # a long prompt between two blocks
        {"name": "norm_prompt", "op": "norm", "m": 8192, "h": 4096, "branch": "bf16", "post": True, "gate": "row", "out": "e4m3"},
        # Llama-8B's down projection quantized at load
        {"name": "quantize_weight", "op": "quantize", "m": 4096, "k": 14336, "rows": 128, "type": "bf16", "fmt": "e4m3"},
        # attention output of a short prompt, rows and columns that fill no whole block
        {"name": "quantize_rows", "op": "quantize", "m": 333, "k": 5000, "rows": 1, "type": "f32", "fmt": "e5m2"},
        # the MLP's activation of a decode step of 8 sequences
        {"name": "swiglu_batch", "op": "swiglu", "m": 8, "k": 14336, "type": "bf16", "fmt": "e4m3"},
        # and of a long prompt
        {"name": "swiglu_prompt", "op": "swiglu", "m": 8192, "k": 14336, "type": "bf16", "fmt": "e4m3"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "product", "norm", "norm", "quantize", "swiglu"])
    fmt = rng.choice(["e4m3", "e4m3", "e5m2"])
    if op == "product":
        while True:  # any row count, output width and depth; a depth of any size is kept in rows of 16-byte pitch
            m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 16, 28672), _log_int(rng, 64, 28672)
            if m * n * k <= 8192 * 28672 * 4096:
                return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "f32"]), "xf": fmt,
                        "wf": rng.choice(["e4m3", "e4m3", "e5m2"])}
    if op == "norm":
        return {"op": op, "m": _log_int(rng, 1, 8192), "h": _log_int(rng, 64, 8192),
                "branch": rng.choice(["bf16", "f32"]), "post": rng.random() < 0.5,
                "gate": rng.choice(["none", "row", "full"]), "out": rng.choice(["bf16", "e4m3", "e4m3", "e5m2"])}
    if op == "quantize":
        return {"op": op, "m": _log_int(rng, 1, 8192), "k": _log_int(rng, 16, 14336), "rows": rng.choice([1, 128]),
                "type": rng.choice(["bf16", "f32"]), "fmt": fmt}
    return {"op": op, "m": _log_int(rng, 1, 8192), "k": _log_int(rng, 16, 14336),
            "type": rng.choice(["bf16", "f32"]), "fmt": fmt}


_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_MAX = {"e4m3": E4M3_MAX, "e5m2": E5M2_MAX}


def _up(n, to):
    return -(-n // to) * to


def _activations(g, m, k):
    """Rows as a decoder has them: unit normal, a few channels far larger."""
    x = torch.randn((m, k), generator=g, device="cuda")
    loud = torch.rand((k,), generator=g, device="cuda") < 0.004
    return torch.where(loud, 30.0, 1.0) * x


def _codes(x, rows, fmt):
    """An operand as the caller of the product holds it: codes in rows of 16-byte pitch, f32 scales."""
    m, k = x.shape
    pad = torch.zeros((_up(m, rows), _up(k, GROUP)), device="cuda")
    pad[:m, :k] = x
    t = pad.view(_up(m, rows) // rows, rows, -1, GROUP)
    top = t.abs().amax((1, 3), keepdim=True)
    s = torch.where(top > 0, top / _MAX[fmt], 1.0)
    q = (t / s).clamp(-_MAX[fmt], _MAX[fmt]).view_as(pad)[:m].to(_F8[fmt]).view(torch.uint8)
    kept = torch.zeros((m, _up(k, 16)), dtype=torch.uint8, device="cuda")
    kept[:, :k] = q[:, :k]
    return kept[:, :k], s.view(s.shape[0], s.shape[2]).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "product":
        s["x"], s["sx"] = _codes(_activations(g, case["m"], case["k"]), 1, case["xf"])
        w = 0.02 * torch.randn((case["n"], case["k"]), generator=g, device="cuda")
        s["w"], s["sw"] = _codes(w, GROUP, case["wf"])
    elif case["op"] == "norm":
        m, h = case["m"], case["h"]
        s["branch"] = _activations(g, m, h).to(_TYPES[case["branch"]])
        s["residual"] = (3 * _activations(g, m, h)).to(torch.bfloat16)
        s["pre"] = 1 + 0.1 * torch.randn((h,), generator=g, device="cuda")
        s["gain"] = 1 + 0.1 * torch.randn((h,), generator=g, device="cuda") if case["post"] else None
        s["mult"] = None
        if case["gate"] != "none":
            shape = (m, h) if case["gate"] == "full" else (h,)
            s["mult"] = torch.rand(shape, generator=g, device="cuda").to(torch.bfloat16)
        s["scale"] = 0.22
    elif case["op"] == "quantize":
        s["x"] = _activations(g, case["m"], case["k"]).to(_TYPES[case["type"]])
    else:
        both = 2 * _activations(g, case["m"], 2 * case["k"])
        s["both"] = both.to(_TYPES[case["type"]])
    return s


# ------------------------------------------------------------------ the plain forms, in 32 bits --
def _spread(scales, rows, m, k):
    """One scale per element from one per block."""
    return scales.repeat_interleave(rows, 0)[:m].repeat_interleave(GROUP, 1)[:, :k]


def _plain_blocks(x, rows, fmt):
    m, k = x.shape
    pad = torch.nn.functional.pad(x, (0, _up(k, GROUP) - k, 0, _up(m, rows) - m))
    top = pad.view(pad.shape[0] // rows, rows, -1, GROUP).abs().amax((1, 3))
    s = torch.where(top > 0, top / _MAX[fmt], 1.0)
    q = (x / _spread(s, rows, m, k)).clamp(-_MAX[fmt], _MAX[fmt])
    return q.to(_F8[fmt]), s


def _plain_norm(x, gain):
    return x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * gain


def _plain(s):
    if s["op"] == "product":
        m, n, k = s["m"], s["n"], s["k"]
        x = s["x"].view(_F8[s["xf"]]).float() * _spread(s["sx"], 1, m, k)
        w = s["w"].view(_F8[s["wf"]]).float() * _spread(s["sw"], GROUP, n, k)
        return (x @ w.T).to(_TYPES[s["out"]])
    if s["op"] == "norm":
        u = s["branch"].float()
        if s["gain"] is not None:
            u = _plain_norm(u, s["gain"])
        if s["mult"] is not None:
            u = u * s["mult"].float()
        y = (s["residual"].float() + s["scale"] * u).to(torch.bfloat16)
        h = _plain_norm(y.float(), s["pre"])
        return (y, h.to(torch.bfloat16)) if s["out"] == "bf16" else (y,) + _plain_blocks(h, 1, s["out"])
    if s["op"] == "quantize":
        return _plain_blocks(s["x"].float(), s["rows"], s["fmt"])
    gate, up = s["both"].float().split(s["k"], 1)
    return _plain_blocks(gate * torch.sigmoid(gate) * up, 1, s["fmt"])


# ------------------------------------------------------------------------ the framework's calls --
def _own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from reng import fp8, gemm, norm
    fmts = {"e4m3": fp8.Fp8Format.E4M3, "e5m2": fp8.Fp8Format.E5M2}
    if s["op"] == "product":
        return gemm.gemm_fp8_blocks(s["x"], s["sx"], s["w"], s["sw"], dtype=_TYPES[s["out"]],
                                    x_fmt=fmts[s["xf"]], w_fmt=fmts[s["wf"]])
    if s["op"] == "norm":
        if s["out"] == "bf16":
            return norm.block_norm(s["residual"], s["branch"], post_gain=s["gain"], gate=s["mult"], scale=s["scale"],
                                   pre_gain=s["pre"], eps=EPS)
        y, q, sc = norm.block_norm_fp8(s["residual"], s["branch"], post_gain=s["gain"], gate=s["mult"],
                                       scale=s["scale"], pre_gain=s["pre"], eps=EPS, fmt=fmts[s["out"]])
        return y, q.view(_F8[s["out"]]), sc
    if s["op"] == "quantize":
        q, sc = fp8.quantize_blocks(s["x"], s["rows"], fmts[s["fmt"]])
    else:
        q, sc = fp8.swiglu_quantize(s["both"], fmts[s["fmt"]])
    return q.view(_F8[s["fmt"]]), sc


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size = {"bf16": 2, "f32": 4}
    m = case["m"]
    if case["op"] == "product":
        n, k = case["n"], case["k"]
        kb = _up(k, GROUP) // GROUP
        return {"bytes": m * k + n * k + 4 * kb * (m + _up(n, GROUP) // GROUP) + m * n * size[case["out"]],
                "flops": 2 * m * n * k}
    if case["op"] == "norm":
        h = case["h"]
        gate = {"none": 0, "row": 2 * h, "full": 2 * m * h}[case["gate"]]
        out = 2 * m * h if case["out"] == "bf16" else m * h + 4 * m * (_up(h, GROUP) // GROUP)
        return {"bytes": m * h * (size[case["branch"]] + 2 + 2) + gate + 4 * h * (2 if case["post"] else 1) + out,
                "flops": m * h * (14 if case["post"] else 10)}
    k = case["k"]
    kb = _up(k, GROUP) // GROUP
    if case["op"] == "quantize":
        rows = case["rows"]
        return {"bytes": m * k * (size[case["type"]] + 1) + 4 * kb * (_up(m, rows) // rows), "flops": 3 * m * k}
    return {"bytes": m * k * (2 * size[case["type"]] + 1) + 4 * kb * m, "flops": 8 * m * k}


# ----------------------------------------------------- the definitions in 64 bits, on their own --
def _values(fmt):
    """The value of each of a format's 256 codes."""
    mant, bias = (3, 7) if fmt == "e4m3" else (2, 15)
    code = torch.arange(256, device="cuda")
    field, frac = (code & 127) >> mant, (code & ((1 << mant) - 1)).double() / (1 << mant)
    size = torch.where(field > 0, torch.ldexp(1 + frac, field - bias), torch.ldexp(frac, torch.full_like(field, 1 - bias)))
    return torch.where(code > 127, -size, size)


def _nearest(v, fmt):
    """v rounded to the nearest value of the format, ties to even, no further than its largest."""
    mant, low = (3, -6) if fmt == "e4m3" else (2, -14)
    e = torch.frexp(v)[1] - 1
    step = torch.ldexp(torch.ones_like(v), e.clamp(min=low) - mant)
    return (torch.round(v / step) * step).clamp(-_MAX[fmt], _MAX[fmt])


def _exact_blocks(x, rows, fmt):
    m, k = x.shape
    out, scales = torch.empty_like(x), torch.empty((_up(m, rows) // rows, _up(k, GROUP) // GROUP), dtype=torch.float64, device="cuda")
    for b in range(scales.shape[1]):
        part = x[:, b * GROUP:(b + 1) * GROUP]
        top = part.abs().amax(1)
        if rows > 1:
            top = torch.nn.functional.pad(top, (0, _up(m, rows) - m)).view(-1, rows).amax(1)
        s = torch.where(top > 0, top / _MAX[fmt], 1.0)
        scales[:, b] = s
        out[:, b * GROUP:(b + 1) * GROUP] = _nearest(part / s.repeat_interleave(rows)[:m, None], fmt)
    return out, scales


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        x, w = _values(case["xf"])[s["x"].long()], _values(case["wf"])[s["w"].long()]
        for b in range(s["sx"].shape[1]):
            cols = slice(b * GROUP, (b + 1) * GROUP)
            x[:, cols] *= s["sx"][:, b:b + 1].double()
            w[:, cols] *= s["sw"][:, b].double().repeat_interleave(GROUP)[:case["n"], None]
        return torch.matmul(x, w.T)
    if case["op"] == "norm":
        u = s["branch"].double()
        if s["gain"] is not None:
            u = s["gain"].double() * u / (u.square().mean(1, keepdim=True) + EPS).sqrt()
        if s["mult"] is not None:
            u = s["mult"].double() * u
        y = s["residual"].double() + s["scale"] * u
        kept = y.to(torch.bfloat16).double()  # the next norm reads the residual as it is stored
        h = s["pre"].double() * kept / (kept.square().mean(1, keepdim=True) + EPS).sqrt()
        return (y, h) if case["out"] == "bf16" else (y,) + _exact_blocks(h, 1, case["out"])
    if case["op"] == "quantize":
        return _exact_blocks(s["x"].double(), case["rows"], case["fmt"])
    g, u = s["both"][:, :case["k"]].double(), s["both"][:, case["k"]:].double()
    return _exact_blocks(g * u / (1 + torch.exp(-g)), 1, case["fmt"])
