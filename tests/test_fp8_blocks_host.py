"""What the 8-bit block operators refuse before touching a device, and calls of
no rows (CPU only)."""
import ctypes as C

import pytest
import torch

INVAL = -1


def last(L):
    return L.reng_last_error().decode()


@pytest.fixture
def L(reng_lib):
    return reng_lib.lib()


GOOD_Q = dict(x=4096, type=0, rows=4, cols=256, ldx=256, block_rows=1, fmt=0, codes=8192, ldc=256, scales=16384, lds=2,
              stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(rows=-1), "rows >= 0"), (dict(cols=0), "cols in [1"), (dict(type=2), "element type"), (dict(fmt=2), "format"),
    (dict(block_rows=64), "block_rows"), (dict(ldx=255), "pitch"), (dict(ldc=255), "pitch"), (dict(lds=1), "pitch"),
    (dict(rows=1 << 41), "2^40"), (dict(ldx=1 << 41), "2^40"), (dict(rows=1 << 30, ldx=1 << 20), "2^40"),
    (dict(x=None), "NULL"), (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(x=4097), "aligned"),
    (dict(scales=16386), "aligned"), (dict(x=4098, type=1), "aligned")])
def test_quantize_blocks_refuses(L, change, word):
    a = {**GOOD_Q, **change}
    assert L.reng_fp8_quantize_blocks(*a.values()) == INVAL
    assert last(L).startswith("reng_fp8_quantize_blocks: ") and word in last(L)


@pytest.mark.parametrize("change,word", [(dict(up=None), "NULL"), (dict(up=8193), "aligned"), (dict(cols=0), "cols"),
                                         (dict(fmt=-1), "format")])
def test_swiglu_quantize_refuses(L, change, word):
    a = {**dict(gate=4096, up=8192, type=0, rows=4, cols=256, ldx=512, fmt=0, codes=8192, ldc=256, scales=16384, lds=2,
                stream=None), **change}
    assert L.reng_fp8_swiglu_quantize(*a.values()) == INVAL
    assert last(L).startswith("reng_fp8_swiglu_quantize: ") and word in last(L)


GOOD_G = dict(x=4096, ldx=256, sx=8192, ldsx=2, xf=0, w=16384, ldw=256, sw=32768, ldsw=2, wf=0, M=4, N=300, K=256,
              y=65536, yt=0, ldy=300, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(M=-1), "M >= 0"), (dict(N=0), "N >= 1"), (dict(K=0), "K >= 1"), (dict(M=(1 << 30) + 1), "2^30"),
    (dict(xf=2), "format"), (dict(wf=-1), "format"), (dict(yt=2), "output type"), (dict(ldx=240), "pitch"),
    (dict(ldw=240), "pitch"), (dict(ldsx=1), "pitch"), (dict(ldsw=1), "pitch"), (dict(ldy=299), "pitch"),
    (dict(x=None), "NULL"), (dict(sx=None), "NULL"), (dict(w=None), "NULL"), (dict(sw=None), "NULL"),
    (dict(y=None), "NULL"), (dict(x=4104), "16"), (dict(w=16385), "16"), (dict(ldx=264), "16"), (dict(ldw=260), "16"),
    (dict(sx=8194), "aligned"), (dict(sw=32769), "aligned"), (dict(y=65537), "aligned"),
    (dict(y=65538, yt=1), "aligned")])
def test_product_refuses(L, change, word):
    a = {**GOOD_G, **change}
    assert L.reng_gemm_fp8_blocks(*a.values()) == INVAL
    assert last(L).startswith("reng_gemm_fp8_blocks: ") and word in last(L)


def desc(reng_lib, **change):
    d = reng_lib.BlockNormDesc()
    for k, v in {**dict(branch=4096, residual=8192, y=16384, h=32768, h_scales=65536, rows=4, cols=256, ld_branch=256,
                        ld_residual=256, ld_y=256, ld_h=256, ld_scales=2, out=reng_lib.RENG_NORM_E4M3, scale=1.0,
                        eps=1e-5), **change}.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,word", [
    (dict(rows=-1), "rows >= 0"), (dict(cols=0), "cols in [1"), (dict(residual_type=2), "element type"),
    (dict(branch_type=-1), "element type"), (dict(gate=4096, ld_gate=256, gate_type=5), "element type"),
    (dict(out=5), "output kind"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(scale=float("inf")), "scale"), (dict(branch=None, out=0), "nothing to do"),
    (dict(branch=None, gate=4096), "without a branch"), (dict(branch=None, post_gain=4096), "without a branch"),
    (dict(ld_residual=255), "pitch"), (dict(ld_branch=255), "pitch"), (dict(ld_y=255), "pitch"),
    (dict(gate=4096, ld_gate=255), "pitch"), (dict(ld_h=255), "pitch"), (dict(ld_scales=1), "pitch"),
    (dict(residual=None), "NULL"), (dict(y=None), "NULL"), (dict(h=None), "NULL"), (dict(h_scales=None), "NULL"),
    (dict(branch=4097), "aligned"), (dict(post_gain=4098), "aligned"), (dict(pre_gain=4097), "aligned"),
    (dict(h_scales=65538), "aligned"), (dict(gate=4097, ld_gate=0), "aligned")])
def test_block_norm_refuses(L, reng_lib, change, word):
    d = desc(reng_lib, **change)
    assert L.reng_block_norm(C.byref(d), None) == INVAL
    assert last(L).startswith("reng_block_norm: ") and word in last(L)
    assert L.reng_block_norm(None, None) == INVAL


def test_no_rows_need_no_buffers(L, reng_lib):
    assert L.reng_fp8_quantize_blocks(*{**GOOD_Q, "rows": 0, "x": None, "codes": None, "scales": None}.values()) == 0
    assert L.reng_gemm_fp8_blocks(*{**GOOD_G, "M": 0, "x": None, "sx": None, "y": None}.values()) == 0
    d = desc(reng_lib, rows=0, residual=None, branch=None, h=None, h_scales=None, y=None)
    assert L.reng_block_norm(C.byref(d), None) == 0


def test_python_refuses_what_is_not_a_device_matrix(reng_lib):
    from reng import fp8, gemm, norm
    x = torch.zeros(4, 256)
    u8 = torch.zeros(4, 256, dtype=torch.uint8)
    for call in (lambda: fp8.quantize_blocks(x), lambda: fp8.swiglu_quantize(x), lambda: norm.block_norm(x),
                 lambda: norm.block_norm_fp8(x, x), lambda: gemm.gemm_fp8_blocks(u8, x[:, :2], u8, x[:1, :2])):
        with pytest.raises(ValueError, match="CUDA device"):
            call()


def test_block_norm_desc_layout(reng_lib):
    """Field order and offsets of the ctypes mirror against the header's struct."""
    import os
    import re
    from conftest import ROOT
    text = open(os.path.join(ROOT, "include", "reng_cuda.h")).read()
    body = re.search(r"typedef struct reng_block_norm_desc \{(.*?)\} reng_block_norm_desc;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n for n in re.findall(r"(\w+)\s*[,;]", body)]
    assert names == [f[0] for f in reng_lib.BlockNormDesc._fields_]
    rs = open(os.path.join(ROOT, "include", "reng_cuda_ffi.rs")).read()
    rs = re.search(r"pub struct reng_block_norm_desc \{(.*?)\n\}", rs, re.S).group(1)
    assert re.findall(r"pub (\w+):", rs) == names
    assert C.sizeof(reng_lib.BlockNormDesc) == 8 * 8 + 8 * 8 + 6 * 4


# ---- the engine's block-scaled weights ----

def test_the_switch_knows_blocks():
    from reng.model import fp8_switch
    assert fp8_switch("blocks") == ("e4m3", "blocks") and fp8_switch("e4m3:blocks", True).backoff == 1.0
    for v in ("e5m2:blocks", "blocks,backoff=0.5", "block"):
        with pytest.raises(ValueError):
            fp8_switch(v)


def test_the_quantize_tool_refuses_blocks():
    from reng.cli import UsageError, fp8_report_line, parse_fp8_quantize, plan_weights
    for argv, env in ((["m", "--fp8", "blocks"], None), (["m"], "blocks")):
        with pytest.raises(UsageError, match="blocks"):
            parse_fp8_quantize(argv, env=env)
    assert "128 x 128" in fp8_report_line(None, None, ("e4m3", "blocks"))
    assert [plan_weights(f) for f in (None, ("e4m3", "pcs"), ("e4m3", "blocks"))] == ["bf16", "fp8", "fp8_blocks"]


def test_blocks_of_another_format_are_refused():
    from reng.config import LlamaConfig
    from reng.model import Engine
    from reng.weights import random_weights
    cfg = LlamaConfig(hidden_size=64, intermediate_size=64, num_hidden_layers=1, num_attention_heads=4,
                      num_key_value_heads=2, head_dim_=16, vocab_size=64)
    with pytest.raises(ValueError, match="e4m3"):
        Engine(cfg, random_weights(cfg), fp8=("e5m2", "blocks"))


def test_the_commands_take_blocks():
    from reng import cli
    argv = ["m", "o", "2", "--fp8", "7"]
    assert cli.parse_generate(argv, env="blocks")["fp8"] == ("e4m3", "blocks")
    assert cli.parse_generate(["m", "o", "2", "7"], env="e4m3,blocks")["fp8"] == ("e4m3", "blocks")
    with pytest.raises(cli.UsageError, match="do not shard"):
        cli.parse_tp(["m", "8", "1", "--modules", "0,1"], env="blocks")


def test_the_plan_counts_block_scales():
    from reng.config import LlamaConfig
    from reng.plan import CachePlan
    cfg = LlamaConfig(hidden_size=256, intermediate_size=400, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim_=64, vocab_size=1024)
    p = CachePlan.new(cfg, weights="fp8_blocks")
    codes = 2 * (512 * 256 + 256 * 256 + 800 * 256 + 256 * 400)
    scales = 2 * (4 * 2 + 2 * 2 + 7 * 2 + 2 * 4)
    assert p.weight_bytes == codes + 4 * scales + 2 * 1024 * 256 * 2
    q = CachePlan.new(cfg, weights="fp8")
    rows = (p.transient_bytes_at(64) - q.transient_bytes_at(64)) / (400 + 4 * 4 + 2 * 800 + 2 * 256 - 2 * 400)
    assert rows == int(rows) and rows >= 256


def test_blocks_do_not_shard(reng_lib):
    import ctypes as C
    from reng import _lib
    d = _lib.ModelDesc(hidden=256, inter=512, n_layers=1, n_heads=4, n_kv_heads=2, head_dim=64, vocab=256, eps=1e-5,
                       attn_scale=0.125, weights=_lib.RENG_WEIGHTS_FP8_BLOCKS, batch=1, capacity=64, tp_world=2)
    out, layer, one = C.c_void_p(), _lib.LayerWeights(), C.c_void_p(16)
    with pytest.raises(Exception, match="do not shard"):
        _lib.call("reng_model_create", C.byref(d), C.byref(layer), one, one, one, one, one, _lib.RENG_MEM_HOST,
                  C.byref(out))
    d.weights, d.tp_world = 3, 1
    with pytest.raises(Exception, match="unknown weight format"):
        _lib.call("reng_model_create", C.byref(d), C.byref(layer), one, one, one, one, one, _lib.RENG_MEM_HOST,
                  C.byref(out))
