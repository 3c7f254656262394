"""The package imports where its libraries are missing or cannot be loaded (built for another torch, or an older build); a call that needs one
says what is wrong."""
import os
import shutil
import subprocess
import sys

import pytest

import adcdiff

PACKAGE = os.path.dirname(os.path.abspath(adcdiff._lib.__file__))
PROGRAM = """
import torch
import adcdiff
from adcdiff import ops
adcdiff.DiffusionModel(dict(input_dim=128, hidden_dim=128, output_dim=128, num_timesteps=10))
assert "groupnorm_silu" in adcdiff.torch_ops.names()
for call in (lambda: ops.row_norm(torch.zeros(2, 8)), lambda: ops.grad_norm([torch.zeros(2)])):
    try:
        call()
        raise SystemExit("no error")
    except adcdiff.AdcdiffError as e:
        print(e)
"""


def _tree(tmp_path):
    pkg = tmp_path / os.path.basename(PACKAGE)
    shutil.copytree(PACKAGE, pkg, ignore=shutil.ignore_patterns("build", "__pycache__", "*.so", "csrc"))
    shutil.copy(os.path.join(os.path.dirname(PACKAGE), "adcdiff.py"), tmp_path)
    return pkg


def _run(tmp_path):
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=str(tmp_path), capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]
    return done.stdout


def test_libraries_missing(tmp_path):
    _tree(tmp_path)
    assert "is missing" in _run(tmp_path)


@pytest.mark.parametrize("broken", ["libadcdiff.so", "libadcdiff_torch.so"])
def test_library_that_does_not_load(tmp_path, broken):
    pkg = _tree(tmp_path)
    for name in ("libadcdiff.so", "libadcdiff_torch.so"):
        if name != broken:
            os.symlink(os.path.join(PACKAGE, name), pkg / name)
    (pkg / broken).write_bytes(b"not a library")
    assert broken in _run(tmp_path)


def test_library_of_an_older_build(tmp_path):
    """one without the entry points that the package binds"""
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    pkg = _tree(tmp_path)
    (tmp_path / "old.c").write_text("int adcdiff_abi_version(void) { return 3; }\n")
    subprocess.run([gcc, "-shared", "-fPIC", str(tmp_path / "old.c"), "-o", str(pkg / "libadcdiff.so")], check=True)
    os.symlink(os.path.join(PACKAGE, "libadcdiff_torch.so"), pkg / "libadcdiff_torch.so")
    assert "libadcdiff.so" in _run(tmp_path)
