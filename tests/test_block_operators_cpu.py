"""Refusals, shape rules and host-side checks of the gated residual norms, the gradient norm and the 8-bit integer layer.
No kernel is launched here: every call ends on the host."""
import ctypes as C

import pytest
import torch

import adcdiff
from adcdiff import _lib, ops

OPERATORS = ("residual_norm", "residual_norm_backward", "grad_norm", "clip_grad_norm_", "clip_grad_norm_out", "quantize_rows", "gemm_int8", "linear_int8")


def _message():
    return _lib.load().adcdiff_last_error().decode()


def test_operators_are_registered():
    for n in OPERATORS:
        assert n in adcdiff.torch_ops.names()
        assert str(getattr(torch.ops.adcdiff, n).default._schema).startswith("adcdiff::" + n)


def test_fake_rules():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        h, x = torch.empty(6, 40, device="cuda", dtype=torch.bfloat16), torch.empty(6, 40, device="cuda")
        xn, y, st = torch.ops.adcdiff.residual_norm(h, x, None, None, None, None, None, 1, 2, 1.0, 1e-6, True, True)
        assert (xn.dtype, y.dtype, tuple(st.shape)) == (torch.float32, torch.bfloat16, (6, 4))
        got = torch.ops.adcdiff.residual_norm_backward(h, x, None, None, None, None, None, st, xn, y, 1, 2, 1.0, 1e-6, [True, True] + 5 * [False])
        assert [(t.shape, t.dtype) for t in got] == [(h.shape, h.dtype), (x.shape, x.dtype)]
        q, s = torch.ops.adcdiff.quantize_rows(torch.empty(5, 33, device="cuda"))
        assert tuple(q.shape) == (5, 33) and q.stride() == (48, 1) and q.dtype == torch.int8 and tuple(s.shape) == (5,)
        assert torch.ops.adcdiff.gemm_int8(q, s, q, s, None, None, 0, 1).dtype == torch.bfloat16
        assert tuple(torch.ops.adcdiff.linear_int8(x, torch.empty(7, 40, device="cuda", dtype=torch.int8), s, None, None, 1, 0).shape) == (6, 7)
        assert torch.ops.adcdiff.clip_grad_norm_([x, h], 1.0, 2).shape == ()


def test_no_cpu_path():
    x = torch.zeros(4, 32)
    i8, s = torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: ops.residual_norm(x, x, pre_norm="rms"), lambda: ops.row_norm(x), lambda: ops.grad_norm([x]), lambda: ops.clip_grad_norm_([x], 1.0),
                 lambda: ops.quantize_rows(x), lambda: ops.gemm_int8(i8, s, i8, s), lambda: ops.linear_int8(x, i8, s)):
        with pytest.raises(adcdiff.AdcdiffError):
            call()


def test_bad_names_and_numbers():
    x = torch.zeros(4, 32)
    with pytest.raises(ValueError):
        ops.residual_norm(x, x, post_norm="batch")
    with pytest.raises(ValueError):
        ops.row_norm(x, norm=None)
    with pytest.raises(ValueError):
        ops.grad_norm([x], norm_type=3)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([x], bad)
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([x], 1.0, out=[])
    with pytest.raises(TypeError):
        ops.grad_norm([1.0])
    with pytest.raises(ValueError):
        ops.gemm_int8(x, x, x, x, out_dtype="fp16")


def test_empty_list_has_norm_zero():
    assert float(ops.grad_norm([])) == 0.0 and float(ops.clip_grad_norm_([], 1.0)) == 0.0


def _norm_args(**over):
    a = _lib.ResidualNormArgs()
    given = dict(M=4, D=32, dtype=1, stream_dtype=0, gate_dtype=1, post_norm=1, pre_norm=1, gate_rows=2, h=4096, ldh=32, x=8192, ldx=32, gate=16384, ldg=32,
                 residual_scale=1.0, eps=1e-6, x_new=32768, ldx_new=32, y=65536, ldy=32)
    given.update(over)
    for k, v in given.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over, words", [
    (dict(D=0), "columns"), (dict(D=8193), "columns"), (dict(M=-1), "rows"), (dict(dtype=2), "types"), (dict(gate_dtype=7), "types"),
    (dict(post_norm=3), "norms"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(x=None), "null x"), (dict(h=None), "without h"),
    (dict(gate_rows=3), "do not divide"), (dict(gate_rows=0), "do not divide"), (dict(ldh=31), "pitch"), (dict(ldx=5), "pitch"), (dict(ldg=16), "pitch"),
    (dict(ldy=31), "pitch"), (dict(y=None), "pre norm"), (dict(pre_norm=0), "pre norm"), (dict(pre_norm=0, y=None, x_new=None), "no output"),
    (dict(post_norm=0, post_weight=4096), "without its norm"), (dict(stats=4100), "16-byte"),
])
def test_residual_norm_refusals(over, words):
    assert _lib.load().adcdiff_residual_norm(C.byref(_norm_args(**over)), None) == -1
    assert words in _message()


@pytest.mark.parametrize("over, grads, code, words", [
    ({}, dict(), -1, "no incoming"), (dict(pre_norm=0), dict(d_y=4096, ld_d_y=32), -1, "without a pre norm"), ({}, dict(d_y=4096, ld_d_y=32), -1, "statistics"),
    (dict(stats=4096, gate=None), dict(d_y=4096, ld_d_y=32, gate=4096, ld_gate=32), -1, "did not have"),
    (dict(stats=4096), dict(d_y=4096, ld_d_y=16), -1, "pitch"), (dict(stats=4096), dict(d_y=4096, ld_d_y=32, x=4096, ld_x=32), -4, "workspace"),
])
def test_residual_norm_backward_refusals(over, grads, code, words):
    g = _lib.ResidualNormGrads()
    for k, v in grads.items():
        setattr(g, k, v)
    assert _lib.load().adcdiff_residual_norm_backward(C.byref(_norm_args(**over)), C.byref(g), None, 0, None) == code
    assert words in _message()


def _table(*rows):
    t = (_lib.GradTensor * max(1, len(rows)))()
    for e, (grad, out, numel, dtype, out_dtype) in zip(t, rows):
        e.grad, e.out, e.numel, e.dtype, e.out_dtype = grad, out, numel, dtype, out_dtype
    return t, len(rows)


@pytest.mark.parametrize("rows, words", [
    ([(4096, 4096, 64, 0, 0), (4096, 4096, 64, 0, 0)], "overlaps"),            # the same tensor twice
    ([(4096, 4096, 64, 0, 0), (4096 + 252, 4096 + 252, 8, 0, 0)], "overlaps"),  # the last element shared
    ([(4096, 4096, 64, 0, 0), (8192, 4096 + 128, 64, 1, 0)], "overlaps"),       # one tensor's output in another's gradient
    ([(4096, 8192, 64, 0, 0), (16384, 4096, 64, 0, 0)], "overlaps"),            # output over a gradient that is read
    ([(4096, 4096, 64, 1, 0)], "overlaps"),                                     # bf16 widened onto itself
    ([(4097, 4097, 4, 0, 0)], "aligned"), ([(4096, 4096, -1, 0, 0)], "elements"), ([(4096, 4096, 4, 5, 0)], "types"), ([(None, None, 4, 0, 0)], "null"),
])
def test_clip_refusals(rows, words):
    t, n = _table(*rows)
    assert _lib.load().adcdiff_clip_grad_norm(t, n, 2, 1.0, 4096, None, 0, None) == -1
    assert words in _message()


def test_clip_accepts_neighbours_and_reading_twice():
    lib = _lib.load()
    neighbours, n = _table((4096, 4096, 64, 0, 0), (4352, 4352, 64, 0, 0), (8192, 16384, 8, 1, 0), (8192, 16416, 8, 1, 0))
    assert lib.adcdiff_clip_grad_norm(neighbours, n, 2, 1.0, 4096, None, 0, None) == -4     # passes every check up to the workspace
    assert "workspace" in _message()
    twice, n = _table((4096, None, 64, 0, 0), (4096, None, 64, 0, 0))
    assert lib.adcdiff_grad_norm(twice, n, 2, 4096, None, 0, None) == -4
    assert lib.adcdiff_grad_norm(twice, n, 1, 4096, None, 0, None) == -1 and "norm type" in _message()
    assert lib.adcdiff_clip_grad_norm(neighbours, 4, 2, -1.0, 4096, None, 0, None) == -1 and "max_norm" in _message()
    assert lib.adcdiff_grad_norm_workspace_bytes(twice, n) == lib.adcdiff_grad_norm_workspace_bytes(neighbours, 2) > 0


def _gemm_args(**over):
    a = _lib.GemmI8Args()
    given = dict(M=4, N=8, K=32, a=4096, lda=32, w=8192, ldw=32, a_scale=4096, w_scale=4096, act=0, out_dtype=1, out=16384, ldo=8)
    given.update(over)
    for k, v in given.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over, words", [
    (dict(K=131072), "K 131072"), (dict(K=0), "K 0"), (dict(N=0), "N 0"), (dict(M=-1), "M -1"), (dict(out_dtype=2), "type"), (dict(act=2), "act"),
    (dict(a=None), "null"), (dict(w_scale=None), "null"), (dict(a=4100), "16-byte"), (dict(lda=40), "16-byte"), (dict(ldw=16), "16-byte"),
    (dict(ldo=7), "pitch"), (dict(residual=4096, ldr=7), "pitch"),
])
def test_gemm_i8_refusals(over, words):
    assert _lib.load().adcdiff_gemm_i8(C.byref(_gemm_args(**over)), None) == -1
    assert words in _message()


def test_linear_i8_refusals():
    lib = _lib.load()
    need = lib.adcdiff_linear_i8_workspace_bytes(4, 32)
    assert need >= 4 * 32 + 4 * 4 and lib.adcdiff_linear_i8_workspace_bytes(4, 0) == 0
    for args, ws, size, code, words in ((dict(), 4096, need - 1, -4, "workspace"), (dict(), None, need, -4, "workspace"), (dict(), 4100, need, -4, "workspace"),
                                        (dict(K=0), 4096, need, -1, "columns"), (dict(act=9), 4096, need, -1, "act"), (dict(w=None), 4096, need, -1, "null")):
        assert lib.adcdiff_linear_i8(4096, 32, 0, C.byref(_gemm_args(**args)), ws, size, None) == code and words in _message()
    assert lib.adcdiff_linear_i8(4096, 31, 0, C.byref(_gemm_args()), 4096, need, None) == -1 and "pitch" in _message()


def test_row_quantiser_refusals():
    lib = _lib.load()
    for args, words in (((4096, 32, 0, -1, 32, 4096, 32, 4096), "rows"), ((4096, 32, 0, 4, 0, 4096, 32, 4096), "columns"), ((4096, 32, 3, 4, 32, 4096, 32, 4096), "type"),
                        ((None, 32, 0, 4, 32, 4096, 32, 4096), "null"), ((4096, 31, 0, 4, 32, 4096, 32, 4096), "pitch"), ((4096, 32, 0, 4, 32, 4096, 31, 4096), "pitch")):
        assert lib.adcdiff_quantize_rows(*args, None) == -1 and words in _message()
    for src, ld_src, M, K, dst, ld_dst in ((4096, 31, 4, 32, 4096, 32), (4096, 32, 4, 32, 4096, 40), (4096, 32, 4, 32, 4100, 32), (None, 32, 4, 32, 4096, 32), (4096, 32, 4, 0, 4096, 32)):
        bad = (_lib.I8Copy * 2)(_lib.I8Copy(4096, 32, 4096, 32, 4, 32), _lib.I8Copy(src, ld_src, dst, ld_dst, M, K))
        assert lib.adcdiff_pitch_rows_i8(bad, 2, None) == -1 and "pitch_rows_i8" in _message()
    assert lib.adcdiff_pitch_rows_i8(None, 1, None) == -1 and lib.adcdiff_pitch_rows_i8(bad, 3, None) == -1


def test_new_structs_match_the_header_layout(tmp_path):
    import os
    import shutil
    import subprocess
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    pairs = [("adcdiff_residual_norm_args", _lib.ResidualNormArgs), ("adcdiff_residual_norm_grads", _lib.ResidualNormGrads),
             ("adcdiff_grad_tensor", _lib.GradTensor), ("adcdiff_gemm_i8_args", _lib.GemmI8Args), ("adcdiff_i8_copy", _lib.I8Copy)]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "adcdiff.h"', 'int main(void) {']
    for cname, ct in pairs:
        lines.append('printf("%s size %%zu\\n", sizeof(%s));' % (cname, cname))
        lines += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f) for f, _ in ct._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ['return 0;', '}']))
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([gcc, "-I", os.path.join(root, "include"), str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in got.strip().splitlines()}
    for cname, ct in pairs:
        assert got[(cname, "size")] == C.sizeof(ct), cname
        for f, _ in ct._fields_:
            assert got[(cname, f)] == getattr(ct, f).offset, (cname, f)
