"""Every kernel of the 8-bit integer product at its edges, whatever the rule would choose there: each is asked for by name.

The kernels share the definition of what follows the exact sum, so their results are the same bits; the 64-bit form (tests/block_reference.py) holds
them to it (at most 10 roundings: conversion, two scales, bias, residual, SiLU's four)."""
import ctypes as C
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

adcdiff = pytest.importorskip("adcdiff")
from adcdiff import _lib, ops  # noqa: E402
import block_reference as ref  # noqa: E402

BF, F = torch.bfloat16, torch.float32
TYPES = {"bf16": BF, "fp32": F}
STEPS = 10


@pytest.fixture
def kernel():
    yield lambda k: _lib.debug_set("gemm_i8_kernel", k)
    _lib.debug_set("gemm_i8_kernel", 0)


def _inputs(M, N, K, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed + M * 31 + N * 17 + K)
    pitch = (K + 15) // 16 * 16

    def codes(rows):          # anything behind K
        return torch.randint(-128, 128, (rows, pitch), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)[:, :K]
    a, w = codes(M), codes(N)
    sa, sw = torch.rand(M, generator=gen, device="cuda") * 0.01 + 1e-3, torch.rand(N, generator=gen, device="cuda") * 0.01 + 1e-3
    return a, sa, w, sw, torch.randn(N, generator=gen, device="cuda"), torch.randn(M, N, generator=gen, device="cuda")


def _check(kernel, k, M, N, K, out, bias, residual, act):
    a, sa, w, sw, b, r = _inputs(M, N, K, 0)
    b, r = b if bias else None, r.to(TYPES[out]) if residual else None
    kernel(k)
    y = ops.gemm_int8(a, sa, w, sw, bias=b, residual=r, act=act, out_dtype=out)
    value, mag = ref.layer(a, sa, w, sw, b, r, act)
    ref.close(y, value, mag, TYPES[out], STEPS)
    kernel(64 if k != 64 else 128)
    assert torch.equal(y, ops.gemm_int8(a, sa, w, sw, bias=b, residual=r, act=act, out_dtype=out))


# 256 x 256 tiles: one, two and more whole K tiles of 128 (the main loop's count is two less, even and odd), columns behind them in every sort, tiles
# that move back inside the matrix by one row or column and by 255, widths that are no multiple of 8
LARGE = [(256, 256, 256), (256, 256, 384), (257, 264, 512), (511, 512, 640), (512, 257, 768), (300, 511, 1152), (769, 263, 257), (256, 520, 271), (258, 300, 272), (400, 259, 383),
         (513, 513, 385), (600, 777, 643), (600, 776, 1000), (300, 1027, 1300), (1030, 290, 2047), (270, 1290, 3001), (1025, 515, 4100)]


@pytest.mark.parametrize("M, N, K", LARGE)
def test_large_tiles(kernel, M, N, K):
    for out, (bias, residual, act) in itertools.product(("fp32", "bf16"), ((True, False, 0), (False, True, 0), (True, False, 1), (True, True, 1))):
        _check(kernel, 256, M, N, K, out, bias, residual, act)


@pytest.mark.parametrize("k", [16, 3216, 32, 64, 128])
@pytest.mark.parametrize("M, N, K", [(1, 1, 1), (3, 17, 15), (16, 16, 128), (17, 33, 129), (33, 40, 255), (63, 65, 256), (64, 64, 384), (65, 63, 385), (127, 129, 511), (129, 127, 640), (130, 263, 1003), (200, 200, 2050)])
def test_small_tiles(kernel, M, N, K, k):
    for out, (bias, residual, act) in zip(("fp32", "bf16", "fp32", "bf16"), ((True, False, 0), (False, True, 0), (True, False, 1), (True, True, 1))):
        _check(kernel, k, M, N, K, out, bias, residual, act)


@pytest.mark.parametrize("k", [256, 128, 64, 32, 3216, 16])
@pytest.mark.parametrize("out", ["fp32", "bf16"])
@pytest.mark.parametrize("M, N, K", [(257, 259, 300), (511, 264, 512), (700, 515, 300), (256, 256, 512)])
def test_residual_in_place(kernel, M, N, K, out, k):
    """out over the residual (C ABI), at odd pitches and addresses: tiles overlap at the edges, each element is read before it is written once,
    and nothing between the rows is written"""
    for pad in (0, 3):
        _in_place(kernel, M, N, K, pad, out, k)


def _in_place(kernel, M, N, K, pad, out, k):
    a, sa, w, sw, _, _ = _inputs(M, N, K, 1)
    pitch, first = N + pad, pad // 2
    held = torch.randn(M * pitch + 1, device="cuda").to(TYPES[out])
    before, rows = held.clone(), held[first:first + M * pitch].view(M, pitch)[:, :N]
    kernel(64 if k != 64 else 128)
    want = ops.gemm_int8(a, sa, w, sw, residual=rows.contiguous(), act=1, out_dtype=out)
    p = _lib.GemmI8Args()
    p.M, p.N, p.K, p.act, p.out_dtype, p.lda, p.ldw, p.ldr, p.ldo = M, N, K, 1, int(out == "bf16"), a.stride(0), w.stride(0), pitch, pitch
    p.a, p.w, p.a_scale, p.w_scale, p.residual, p.out = (t.data_ptr() for t in (a, w, sa, sw, rows, rows))
    kernel(k)
    _lib.check(_lib.load().adcdiff_gemm_i8(C.byref(p), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(rows, want)
    inside = torch.zeros(held.shape, dtype=torch.bool, device="cuda")
    inside[first:first + M * pitch].view(M, pitch)[:, :N] = True
    assert torch.equal(held[~inside], before[~inside])


def test_rows_apart_and_poison(kernel):
    """codes as columns of a wider matrix, a scale that is NaN, an infinite residual: they stay in their row"""
    gen = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randint(-128, 128, (900, 2048), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
    a, w = wide[:530, 256:256 + 777], wide[530:, 1024:1024 + 777]
    sa, sw = torch.rand(530, generator=gen, device="cuda"), torch.rand(370, generator=gen, device="cuda")
    r = torch.randn(530, 370, generator=gen, device="cuda")
    sa[500] = float("nan")
    r[3, 260] = float("inf")
    value, mag = ref.layer(a, sa, w, sw, None, r, 0)
    for k in (256, 128, 64, 32, 3216, 16):
        kernel(k)
        y = ops.gemm_int8(a, sa, w, sw, residual=r, out_dtype="fp32")
        assert torch.isnan(y[500]).all() and int(torch.isnan(y).sum()) == 370 and float(y[3, 260]) == float("inf")
        keep = torch.isfinite(value)
        ref.close(y[keep], value[keep], mag[keep], F, STEPS)


def test_rule_takes_the_large_kernel(kernel):
    """shapes of ordinary use on the 256 x 256 kernel: the same bits as by name"""
    for M, N, K in ((10384, 1027, 1643), (5300, 2056, 1024), (8192, 2048, 2048)):
        a, sa, w, sw, b, _ = _inputs(M, N, K, 2)
        y = ops.gemm_int8(a, sa, w, sw, bias=b, act=1)
        for k in (256, 128):
            kernel(k)
            assert torch.equal(y, ops.gemm_int8(a, sa, w, sw, bias=b, act=1))
        kernel(0)


def test_names_that_do_not_fit(kernel):
    a, sa, w, sw, _, _ = _inputs(300, 300, 255, 3)
    for k, words in ((256, "256"), (48, "names no kernel")):
        kernel(k)
        with pytest.raises(adcdiff.AdcdiffError, match=words):
            ops.gemm_int8(a, sa, w, sw)
    kernel(0)
    ops.gemm_int8(a, sa, w, sw)
