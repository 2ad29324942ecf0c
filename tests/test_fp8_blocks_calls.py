"""The 8-bit block operators' host side and index arithmetic beyond the
refusals of test_fp8_blocks_host.py (CPU only)."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

HERE = os.path.dirname(os.path.abspath(__file__))


def run_check(tmp_path, name):
    """Compile and run a harness over one of the kernels' headers."""
    if shutil.which("g++") is None:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path / name)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "reciprocating-engine_b200", "csrc"),
                    os.path.join(HERE, name + ".cc"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_a_product_waits_for_the_last_arrivals_of_its_stages(tmp_path):
    """The copy warp's closing waits name every used stage's last fill."""
    assert " bad 0" in run_check(tmp_path, "ring_check")
    src = open(os.path.join(ROOT, "reciprocating-engine_b200", "csrc", "gemm_fp8.cu")).read()
    # both CTAs of a pair take the wait, before the barrier that ends them
    assert 0 < src.index("landed(B_EMPTY)") < src.index("cta_end<PAIR>();")


def test_a_norm_row_of_any_alignment_is_read_alone(tmp_path):
    """Nothing beside a row is read, where another row may be written meanwhile or memory end."""
    assert " bad 0" in run_check(tmp_path, "row_image_check")


def test_python_raises_what_the_status_tells(monkeypatch, reng_lib):
    from reng import gemm
    codes = [reng_lib.RENG_E_TIMEOUT, reng_lib.RENG_OK]

    class Fake:
        def reng_gemm_fp8_blocks_status(self):
            return codes.pop(0)

        def reng_last_error(self):
            return b"gave up"
    monkeypatch.setattr(reng_lib, "lib", Fake)
    with pytest.raises(reng_lib.RengError, match="gave up"):
        gemm.gemm_fp8_blocks_status()
    gemm.gemm_fp8_blocks_status()
    assert not codes


def test_a_stream_of_another_device_is_refused(monkeypatch):
    import torch
    from reng import _tensors

    class Stream:
        device = torch.device("cuda", 1)

    class Tensor:
        device = torch.device("cuda", 0)

        def get_device(self):
            return 0
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
        _tensors.on_stream(Stream(), Tensor(), lambda: pytest.fail("ran"))
    with pytest.raises(ValueError, match="not on a CUDA device"):
        _tensors.on_stream(7, torch.zeros(2, 128), lambda: pytest.fail("ran"))


def test_a_norm_in_place_at_another_pitch_is_refused(reng_lib):
    import ctypes as C
    d = reng_lib.BlockNormDesc(branch=4096, residual=8192, y=8192, rows=4, cols=256, ld_branch=256, ld_residual=256, ld_y=264,
                               out=reng_lib.RENG_NORM_NONE, scale=1.0, eps=1e-5)
    L = reng_lib.lib()
    assert L.reng_block_norm(C.byref(d), None) == reng_lib.RENG_E_INVAL
    assert b"another row pitch" in L.reng_last_error()
