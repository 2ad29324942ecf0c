"""The engine on block-scaled FP8 weights and 8-bit activations
(RENG_WEIGHTS_FP8_BLOCKS): its layers run reng_block_norm,
reng_gemm_fp8_blocks and the two quantizers one after the other.

Two oracles.  At position 0 attention returns v itself, so a whole model of
several layers is a chain of the public operators with nothing in between:
the engine's logits have to be those of the chain's last norm, up to the LM
head's own rounding.  At later positions one layer with an identity o_proj, no
MLP and an LM head that copies shows attention itself, whose 64-bit form gives
the value and a bound.  The operators' own values are
tests/test_fp8_blocks_gpu.py's matter.
"""
import numpy as np
import pytest

from test_decode_gpu import small_cfg

pytestmark = pytest.mark.gpu

U32, U_BF16, U_E4M3 = 2.0 ** -24, 2.0 ** -8, 2.0 ** -4
BLOCKS = ("e4m3", "blocks")


def bf16(a, dev):
    import torch
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int16)).to(dev).view(torch.bfloat16)


def f32(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(dev)


def product(x, sx, *weights):
    """codes times the block-quantized rows of bf16 matrices laid one below the other."""
    import torch
    from reng import fp8, gemm
    w, sw = fp8.quantize_blocks(torch.cat(weights), 128)
    return gemm.gemm_fp8_blocks(x, sx, w, sw, dtype=torch.bfloat16)


def with_gains(w, seed):
    """Norm gains other than ones, and biases of a size that shows."""
    rng = np.random.default_rng(seed)
    for lw in w["layers"]:
        for k in ("g1", "g2"):
            lw[k] = rng.uniform(0.5, 1.5, lw[k].shape).astype(np.float32)
        for k in ("bq", "bk", "bv"):
            if k in lw:
                lw[k] = (0.3 * rng.standard_normal(lw[k].shape)).astype(np.float32)
    w["final_gamma"] = rng.uniform(0.5, 1.5, w["final_gamma"].shape).astype(np.float32)
    return w


def chain_at_zero(cfg, w, ids, dev="cuda"):
    """Every layer at position 0, one public operator after the other; the
    rows that the LM head takes (bf16)."""
    import torch
    from reng import fp8, norm
    nh, nkv, hd = cfg.num_attention_heads, cfg.n_kv_heads(), cfg.head_dim()
    qd, kvd, eps = nh * hd, nkv * hd, cfg.rms_norm_eps
    res = bf16(w["embed"], dev)[torch.from_numpy(np.asarray(ids, np.int64)).to(dev)].contiguous()
    branch = None
    for lw in w["layers"]:
        res, h, s = norm.block_norm_fp8(res, branch, pre_gain=f32(lw["g1"], dev), eps=eps)
        qkv = product(h, s, *(bf16(lw[k], dev) for k in ("wq", "wk", "wv")))
        v = qkv[:, qd + kvd:].float()
        if "bv" in lw:
            v = v + f32(lw["bv"], dev)
        # a lone key has probability 1: attention is v, for each head of its group
        attn = v.to(torch.bfloat16).view(-1, nkv, 1, hd).expand(-1, nkv, nh // nkv, hd).reshape(-1, qd)
        o = product(*fp8.quantize_blocks(attn.contiguous(), 1), bf16(lw["wo"], dev))
        res, h, s = norm.block_norm_fp8(res, o, pre_gain=f32(lw["g2"], dev), eps=eps)
        both = product(h, s, bf16(lw["wg"], dev), bf16(lw["wu"], dev))
        branch = product(*fp8.swiglu_quantize(both), bf16(lw["wd"], dev))
    return norm.block_norm(res, branch, pre_gain=f32(w["final_gamma"], dev), eps=eps)[1].to(torch.bfloat16)


def check_logits(got, h, w, dev="cuda"):
    """Logits of bf16 rows: f32 sums of H products in some order (H half-steps
    of the sum of magnitudes) and one rounding to bf16."""
    import torch
    h, lm = h.double(), bf16(w["lm_head"], dev).double()
    want, size = h @ lm.T, h.abs() @ lm.abs().T
    err = (torch.from_numpy(np.ascontiguousarray(got)).to(dev).double() - want).abs()
    tol = 1.01 * (U_BF16 * want.abs() + h.shape[1] * U32 * size) + 1e-30
    assert bool((err <= tol).all()), "%d logits off, worst %.3g of the bound" % (
        int((err > tol).sum()), float((err / tol).max()))


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("shape", ["even", "odd"])
@pytest.mark.parametrize("B", [1, 8, 24, 130])
def test_a_chain_of_the_operators_at_position_zero(reng_lib, B, shape, bias):
    from reng.model import Engine
    from reng.synth import prompt_ids
    from reng.weights import random_weights
    # odd: widths that leave part of a group, 3 layers, heads of 48
    kw = {} if shape == "even" else dict(hidden_size=240, intermediate_size=400, num_hidden_layers=3,
                                         num_attention_heads=6, num_key_value_heads=2, head_dim_=48)
    cfg = small_cfg(bias=bias, **kw)
    w = with_gains(random_weights(cfg, seed=41, std=0.05), 41)
    e = Engine(cfg, w, batch=B, capacity=32, fp8=BLOCKS)
    ids = prompt_ids(B, cfg.vocab_size, seed=B)
    logits, _ = e.step_logits(ids)
    check_logits(logits, chain_at_zero(cfg, w, ids), w)
    # and as prompts of one token
    for b in sorted({0, B - 1}):
        e.reset(b)
        _, last, allg = e.prefill(b, ids[b:b + 1], last_logits=True, all_logits=True)
        h = chain_at_zero(cfg, w, ids[b:b + 1])
        check_logits(allg, h, w)
        check_logits(last[None], h, w)
    e.close()


def see_through(cfg, seed):
    """One layer whose residual stream after it is x + attention: an identity
    o_proj, no MLP, and an LM head whose row i copies value i.  Scores are of
    the size of 1 (the bound grows with them), the stream and v of a few."""
    from reng.synth import bf16_bits_to_f32, f32_to_bf16_bits
    from reng.weights import random_weights
    w = with_gains(random_weights(cfg, seed=seed, std=0.03), seed)
    h = cfg.hidden_size

    def by8(t):
        return f32_to_bf16_bits(8 * bf16_bits_to_f32(t)).reshape(t.shape)
    assert cfg.q_dim() == h and cfg.vocab_size >= h
    lw = w["layers"][0]
    w["embed"], lw["wv"] = by8(w["embed"]), by8(lw["wv"])
    lw["wo"] = f32_to_bf16_bits(np.eye(h, dtype=np.float32)).reshape(h, h)
    lw["wd"] = np.zeros_like(lw["wd"])
    lm = np.zeros((cfg.vocab_size, h), np.float32)
    lm[:h] = np.eye(h)
    w["lm_head"] = f32_to_bf16_bits(lm).reshape(lm.shape)
    return w


def attention_oracle(cfg, w, ids, qk_norm, dev="cuda"):
    """(logits [T][H], bound) of the see-through layer, from the operators' own
    q/k/v rows; attention and all after it in 64 bits."""
    import torch
    from reng import norm
    from reng.rope import rope_caches_for
    nh, nkv, hd = cfg.num_attention_heads, cfg.n_kv_heads(), cfg.head_dim()
    qd, kvd, T, lw = nh * hd, nkv * hd, len(ids), w["layers"][0]
    x = bf16(w["embed"], dev)[torch.from_numpy(np.asarray(ids, np.int64)).to(dev)].contiguous()
    _, h, s = norm.block_norm_fp8(x, pre_gain=f32(lw["g1"], dev), eps=cfg.rms_norm_eps)
    qkv = product(h, s, *(bf16(lw[k], dev) for k in ("wq", "wk", "wv"))).double()
    if "bq" in lw:
        qkv = qkv + torch.cat([f32(lw[k], dev) for k in ("bq", "bk", "bv")]).double()
    q, k, v = (t.reshape(T, -1, hd).transpose(0, 1) for t in qkv.split([qd, kvd, kvd], dim=1))
    if qk_norm:
        def n(t, g):
            return t / (t.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt() * f32(lw[g], dev).double()
        q, k = n(q, "qn"), n(k, "kn")
    sin, cos = (f32(t, dev).double().reshape(-1, hd)[:T] for t in rope_caches_for(cfg, T))

    def rot(t):
        return t * cos + torch.cat([-t[..., hd // 2:], t[..., :hd // 2]], -1) * sin
    scale = cfg.attention_scale()
    q, k = rot(q) * scale, rot(k)
    k, v = (t.repeat_interleave(nh // nkv, 0) for t in (k, v))
    dead = torch.ones(T, T, dtype=torch.bool, device=dev).triu(1)
    p = (q @ k.transpose(1, 2)).masked_fill(dead, -float("inf")).softmax(-1)
    # q and k are rounded to bf16 once (twice with their norm: the raw rows
    # first, so 2 half-steps each), which moves a score by 2 or 4 half-steps of
    # sum |q k| (|q||k| bounds it) and a probability by twice the largest move
    # in its row, up and down; p is rounded to bf16 in the product with v, v
    # and the output once more; scores and sums in f32 are in the 1.01
    moves = (4 if qk_norm else 2) * U_BF16 * (q.norm(dim=-1) * k.norm(dim=-1).amax(-1, keepdim=True))
    rel = torch.expm1(2 * 1.01 * moves).unsqueeze(-1) + 3 * U_BF16
    a = (p @ v).transpose(0, 1).reshape(T, qd)
    da = (1.01 * rel * (p @ v.abs())).transpose(0, 1).reshape(T, qd)
    # codes of the rounded a: half a step relative, or half of the lowest step
    # 2^-9 of the group's scale; the product and the stream round to bf16
    top = torch.nn.functional.pad(a.abs() + da, (0, -qd % 128)).reshape(T, -1, 128).amax(-1)
    low = (2.0 ** -10 * top / 240).repeat_interleave(128, -1)[:, :qd]
    da = da + 1.01 * (U_E4M3 + U_BF16) * (a.abs() + da) + low
    y = x.double() + a
    dy = da + 1.01 * U_BF16 * (y.abs() + da)
    # the norm at y + e, |e| <= dy: |y + e| lies within |y| (1 -+ m) for
    # m = |dy| / |y| < 1, so r moves by r m / (1 - m) at most, any m below 1
    r = 1 / (y.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt()
    g = f32(w["final_gamma"], dev).double()
    move = dy.norm(dim=-1, keepdim=True) / y.norm(dim=-1, keepdim=True)
    assert float(move.max()) < 1
    want = y * r * g
    bound = r * g * (dy + (y.abs() + dy) * move / (1 - move))
    return want, 1.01 * bound + 2.02 * U_BF16 * (want.abs() + bound)  # h and the logit in bf16


CASES = {
    "gqa": dict(),
    "wide": dict(num_attention_heads=2, num_key_value_heads=1, head_dim_=128),
    "small": dict(num_attention_heads=16, num_key_value_heads=16, head_dim_=16),
}


@pytest.mark.parametrize("case,T", [(c, T) for c in ("gqa", "wide", "small", "bias", "qk_norm")
                                    for T in (2, 9, 70, 300)] + [("gqa", 1100)])  # 1100: two blocks of rows
def test_positions_and_attention(reng_lib, case, T):
    """A prompt's every row, and its last token as a decode step after the
    others, in a slot of its own among others."""
    import torch
    from reng.model import Engine
    from reng.synth import prompt_ids
    cfg = small_cfg(bias=case == "bias", num_hidden_layers=1, **CASES.get(case, {}))
    w = see_through(cfg, 7)
    if case == "qk_norm":
        rng = np.random.default_rng(3)
        for k in ("qn", "kn"):
            w["layers"][0][k] = rng.uniform(0.2, 0.6, cfg.head_dim()).astype(np.float32)
    ids = prompt_ids(T, cfg.vocab_size, seed=T)
    want, bound = attention_oracle(cfg, w, ids, case == "qk_norm")
    H = cfg.hidden_size

    def check(got, rows):
        got = torch.from_numpy(np.ascontiguousarray(got[..., :H])).to(want.device).double().reshape(-1, H)
        err = (got - want[rows]).abs()
        assert bool((err <= bound[rows]).all()), "%d values off, worst %.3g of the bound" % (
            int((err > bound[rows]).sum()), float((err / bound[rows]).max()))
    e = Engine(cfg, w, batch=3, capacity=max(512, T + 1), fp8=BLOCKS)
    check(e.prefill(1, ids, all_logits=True)[2], slice(None))
    e.reset()
    short = max(1, T // 3)
    e.prefill(0, ids[:short])
    e.prefill(2, ids[:T - 1])
    logits, _ = e.step_logits(np.array([ids[short], ids[0], ids[T - 1]], np.uint32))
    check(logits[0], slice(short, short + 1))
    check(logits[1], slice(0, 1))
    check(logits[2], slice(T - 1, T))
    e.close()


@pytest.mark.parametrize("B", [1, 8, 20])
def test_the_captured_step_repeats_the_plain_one(reng_lib, B):
    """decode() replays one captured step; step by step the same ids come from
    the same kernels, twice over."""
    from reng.model import Engine
    from reng.synth import prompt_ids
    from reng.weights import random_weights
    cfg = small_cfg()
    w = random_weights(cfg, seed=43, std=0.05)
    e = Engine(cfg, w, batch=B, capacity=96, fp8=BLOCKS)
    prompts = [prompt_ids(5 + 7 * b % 40, cfg.vocab_size, seed=b) for b in range(B)]

    def start():
        e.reset()
        return [e.prefill(b, p)[0] for b, p in enumerate(prompts)]
    runs = []
    for _ in range(2):
        runs.append(np.asarray(e.decode(start(), 12)))
    ids = np.array(start(), np.uint32)
    steps = []
    for _ in range(12):
        logits, ids = e.step_logits(ids)
        assert np.isfinite(logits).all()
        steps.append(ids)
    e.close()
    assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], np.stack(steps))


def test_the_plan_covers_what_the_engine_allocates(reng_lib):
    from reng.model import Engine
    from reng.plan import CachePlan
    from reng.weights import random_weights
    cfg = small_cfg(hidden_size=512, intermediate_size=1408, num_attention_heads=8, vocab_size=4096)
    w = random_weights(cfg, seed=1)
    used = {}
    for scheme in ("pcs", "blocks"):
        e = Engine(cfg, w, batch=4, capacity=256, fp8=("e4m3", scheme))
        used[scheme] = e.device_bytes()
        e.close()
    plan = CachePlan.new(cfg, batch=4, weights="fp8_blocks")
    need = plan.weight_bytes + plan.cache_bytes_at(256) + plan.transient_bytes_at(256)
    assert used["blocks"] <= need + plan.reserve_bytes and used["blocks"] >= plan.weight_bytes


def test_large_widths(reng_lib):
    """One decode step and one prompt row of two layers of Llama-3.1-8B's
    widths against the chain of operators."""
    from reng.config import llama31_8b
    from reng.model import Engine
    from reng.weights import random_weights, to_host
    cfg = llama31_8b()
    w = random_weights(cfg, seed=5, layers=2, device="cuda")
    cfg.num_hidden_layers = 2
    e = Engine(cfg, w, batch=2, capacity=64, fp8=BLOCKS)
    h = to_host(w)
    ids = np.array([17, 90001], np.uint32)
    check_logits(e.step_logits(ids)[0], chain_at_zero(cfg, h, ids), h)
    e.reset()
    check_logits(e.prefill(1, ids[1:], all_logits=True)[2], chain_at_zero(cfg, h, ids[1:]), h)
    e.close()
