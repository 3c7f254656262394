"""Facts about the sources of the 8-bit integer product that its kernels rely on and no compiler checks."""
import glob
import os
import re
import shutil
import subprocess
import sys

import pytest

import adcdiff

CSRC = os.path.join(os.path.dirname(os.path.abspath(adcdiff._lib.__file__)), "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def test_generated_main_loop_is_what_the_generator_writes(tmp_path):
    out = tmp_path / "i8.inc"
    subprocess.run([sys.executable, os.path.join(CSRC, "gen_w4_mainloop.py"), "--i8", str(out)], check=True)
    assert out.read_text() == open(os.path.join(CSRC, "w4_mainloop_i8.inc")).read()


def test_every_generated_file_is_checked():
    """a third .inc would need a test like the one above"""
    assert sorted(os.path.basename(f) for f in glob.glob(os.path.join(CSRC, "*.inc")) if "stamps" not in f) == ["w4_mainloop.inc", "w4_mainloop_i8.inc"]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_ring_kernels_have_no_scratch(tmp_path):
    """their loops count vmcnt by hand: a spill would add loads to the count"""
    out = tmp_path / "i8.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-S",
                    "--cuda-device-only", "-o", str(out), os.path.join(CSRC, "gemm_i8.hip")], check=True, capture_output=True, timeout=600)
    text = out.read_text()
    ring = re.findall(r"\.amdhsa_kernel (\S*gemm_i8_ring_kernel\S*)\n(.*?)\.end_amdhsa_kernel", text, re.S)
    assert len(ring) == 4
    for name, body in ring:
        assert re.search(r"\.amdhsa_private_segment_fixed_size\s+0\b", body), name
