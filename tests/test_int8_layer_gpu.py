"""The 8-bit integer layer on the GPU: codes equal the float64 definition's exactly, sums are exact integers, the float32 epilogue is held
to its roundings (tests/block_reference.py: at most 10 here, conversion, two scales, bias, residual, SiLU's four)."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

adcdiff = pytest.importorskip("adcdiff")
from adcdiff import ops  # noqa: E402
import block_reference as ref  # noqa: E402

BF, F = torch.bfloat16, torch.float32
TYPES = {"bf16": BF, "fp32": F}
STEPS = 10


def _same_codes(x):
    q, s = ops.quantize_rows(x)
    want_q, want_s = ref.codes(x)
    assert q.dtype == torch.int8 and s.dtype == F and q.shape == x.shape and s.shape == x.shape[:1]
    assert q.data_ptr() % 16 == 0 and (x.shape[0] <= 1 or q.stride(0) % 16 == 0)
    assert torch.equal(q.double(), want_q)
    assert torch.equal(torch.nan_to_num(s), torch.nan_to_num(want_s.float())) and torch.equal(torch.isnan(s), torch.isnan(want_s))
    held = torch.as_strided(q, (q.shape[0], (x.shape[1] + 15) // 16 * 16), (max(q.stride(0), (x.shape[1] + 15) // 16 * 16), 1))
    assert not held[:, x.shape[1]:].any()
    return q, s


@pytest.mark.parametrize("K", [1, 2, 7, 8, 15, 16, 17, 100, 128, 136, 500, 512, 1000, 1003, 2048, 2056, 4095, 4096, 5120, 8192, 8200, 9001])
@pytest.mark.parametrize("dtype", [F, BF])
def test_codes(K, dtype):
    gen = torch.Generator(device="cuda").manual_seed(K)
    for M in (1, 3, 70):
        x = torch.randn(M, K, generator=gen, device="cuda") * torch.exp(3 * torch.randn(M, 1, generator=gen, device="cuda"))
        _same_codes(x.to(dtype))


@pytest.mark.parametrize("M, K", [(2048, 2048), (2050, 1000), (5001, 1300), (70000, 64), (4097, 513)])
@pytest.mark.parametrize("dtype", [F, BF])
def test_codes_of_many_rows(M, K, dtype):
    x = torch.randn(M, K, device="cuda") * torch.exp(3 * torch.randn(M, 1, device="cuda"))
    _same_codes(x.to(dtype))


def test_every_bfloat16_quotient():
    """all pairs of 8-bit significands, over a range of exponents: each row one maximum against every smaller magnitude"""
    sig = torch.arange(128, 256, device="cuda", dtype=torch.float64)
    values = torch.cat([sig * 2.0 ** -e for e in range(0, 9)])
    for shift in (0, 20, -100, 110, 118, -120):
        tops = sig * 2.0 ** shift
        x = (values[None, :] * 2.0 ** shift).expand(128, -1).clone()
        x = torch.where(x <= tops[:, None], x, 0.0)
        x[:, 0] = tops
        x[:, 1::2] *= -1
        assert torch.equal(x.to(BF).double(), x)
        _same_codes(x.to(BF))
        _same_codes(x.to(F))


@pytest.mark.parametrize("dtype", [F, BF])
def test_codes_on_ties(dtype):
    """rows whose quotients are exact halves, and float32 neighbours of halves"""
    rows = []
    for top in (1.0, 254.0, 127.0, 129.0, 1.0078125, 3.96875, 2.0 ** -20, 1e-3, 7.0):
        n = torch.arange(-127, 127, dtype=torch.float64)
        rows.append(torch.cat([(2 * n + 1) / 254.0 * top, torch.tensor([top, -top], dtype=torch.float64)]))
    x = torch.stack(rows).cuda().to(dtype)
    _same_codes(x)
    if dtype == F:
        for step in (-1, 1):
            bits = x.view(torch.int32) + step
            near = bits.view(F).clone()
            near[:, -2:] = x[:, -2:]
            _same_codes(near)


def test_codes_of_extreme_rows():
    x = torch.randn(12, 264, device="cuda")
    x[0] = 0.0
    x[1] *= 1e38
    x[2] *= 1e-38
    x[3] = 1e-45 * torch.randint(-5, 6, (264,), device="cuda").float()
    x[4, 7], x[5, 0], x[6, 263] = float("nan"), float("inf"), -float("inf")
    x[7] = torch.finfo(F).max
    x[8] *= 1e-31
    x[9] = -0.0
    x[10] = torch.where(torch.arange(264, device="cuda") == 9, 1e30, 1e-30)
    q, s = _same_codes(x)
    assert torch.isnan(s[4:7]).all() and not q[4:7].any() and float(s[0]) == 0.0


def test_codes_of_strided_rows():
    held = torch.randn(9, 700, device="cuda")
    for view in (held[:, :333], held[:, 1:640], held[:, 4:516], held[::2, :512], held[:1, 3:20]):
        _same_codes(view)
    assert ops.quantize_rows(held[:0])[0].shape == (0, 700)


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("K, ldq", [(5, 5), (5, 8), (7, 16), (9, 9), (21, 23), (21, 24), (100, 101), (129, 144), (515, 515), (2047, 2048), (4097, 4099), (8195, 8197)])
def test_code_rows_of_any_pitch(K, ldq, dtype):
    """codes at any pitch (C ABI) from rows at odd addresses; zeros up to the next multiple of 16 inside the pitch, the rest untouched"""
    from adcdiff import _lib
    M = 11
    x = torch.randn(M * (K + 3) + 1, device="cuda").to(dtype)[1:].view(M, K + 3)[:, :K]
    want, scale = ops.quantize_rows(x)
    q, got = torch.full((M * ldq + 40,), 99, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    _lib.check(_lib.load().adcdiff_quantize_rows(x.data_ptr(), K + 3, int(dtype == BF), M, K, q.data_ptr(), ldq, got.data_ptr(),
                                                 torch.cuda.current_stream().cuda_stream))
    rows, end = q[:M * ldq].view(M, ldq), min(ldq, (K + 15) // 16 * 16)
    assert torch.equal(rows[:, :K], want) and torch.equal(got, scale)
    assert not rows[:, K:end].any() and bool((rows[:, end:] == 99).all()) and bool((q[M * ldq:] == 99).all())


def test_codes_past_32_bits():
    pitch = (1 << 30) + 16
    held = torch.empty(2 * pitch + 512, device="cuda", dtype=BF)
    far = torch.as_strided(held, (3, 512), (pitch, 1))
    far.copy_(torch.randn(3, 512, device="cuda"))
    a, b = ops.quantize_rows(far), ops.quantize_rows(far.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def _rows16(t, fill=127):
    """t in rows on 16-byte boundaries, with `fill` behind the columns"""
    held = torch.full((t.shape[0], (t.shape[1] + 15) // 16 * 16), fill, dtype=torch.int8, device="cuda")
    held[:, :t.shape[1]] = t
    return held[:, :t.shape[1]]


def _codes(gen, *shape):
    return torch.randint(-128, 128, shape, generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)


def _check(M, N, K, out="fp32", bias=False, residual=False, act=0, pad=True, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + M * 31 + N * 17 + K)
    a, w = _codes(gen, M, K), _codes(gen, N, K)
    sa, sw = torch.rand(M, generator=gen, device="cuda") * 0.01 + 1e-3, torch.rand(N, generator=gen, device="cuda") * 0.01 + 1e-3
    b = torch.randn(N, generator=gen, device="cuda") if bias else None
    r = torch.randn(M, N, generator=gen, device="cuda").to(TYPES[out]) if residual else None
    y = ops.gemm_int8(_rows16(a) if pad else a, sa, _rows16(w) if pad else w, sw, bias=b, residual=r, act=act, out_dtype=out)
    value, mag = ref.layer(a, sa, w, sw, b, r, act)
    ref.close(y, value, mag, TYPES[out], STEPS)


ROWS = [1, 2, 5, 15, 16, 17, 31, 32, 33, 47, 64, 65, 100, 127, 128, 129, 200, 256, 257, 511, 1000]


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("N, K", [(1, 1), (16, 64), (17, 100), (64, 128), (100, 1003), (128, 16), (512, 130), (1000, 512), (48, 4100), (2048, 1024), (260, 2048)])
def test_products(M, N, K):
    _check(M, N, K, "bf16" if (M + N + K) % 2 else "fp32", bias=M % 3 == 0, residual=M % 2 == 0, act=M % 5 == 0)


@pytest.mark.parametrize("K", [1, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 192, 255, 256, 257, 383, 384, 385, 511, 513, 640, 1025, 3001])
@pytest.mark.parametrize("M, N", [(3, 96), (40, 40), (300, 260), (1, 513)])
def test_inner_lengths(M, N, K):
    _check(M, N, K)


@pytest.mark.parametrize("out", ["fp32", "bf16"])
@pytest.mark.parametrize("bias, residual, act", list(itertools.product((False, True), (False, True), (0, 1))))
def test_epilogues(out, bias, residual, act):
    for M, N, K in ((4, 72, 256), (33, 130, 200), (260, 512, 384), (2048, 1024, 512), (1024, 2050, 256)):
        _check(M, N, K, out, bias, residual, act)


@pytest.mark.parametrize("out", ["fp32", "bf16"])
@pytest.mark.parametrize("residual, act", list(itertools.product((False, True), (0, 1))))
@pytest.mark.parametrize("M, N, K", [(8200, 2056, 300), (8192, 2048, 256), (9001, 1800, 643), (16500, 1027, 400), (33000, 257, 513)])
def test_large_products(M, N, K, out, residual, act):
    """tiles that end past the last row and column, columns behind the whole K tiles, outputs on and off 16-byte boundaries"""
    _check(M, N, K, out, True, residual, act)


def test_residual_in_place():
    """out may be the residual itself (C ABI): tiles at the edges overlap, and each element is still read before it is written once"""
    import ctypes as C
    from adcdiff import _lib
    gen = torch.Generator(device="cuda").manual_seed(6)
    for M, N, K in ((8200, 2056, 300), (3000, 1000, 512), (600, 200, 128), (20, 300, 700)):
        a, w = _codes(gen, M, (K + 15) // 16 * 16), _codes(gen, N, (K + 15) // 16 * 16)
        sa, sw = torch.rand(M, generator=gen, device="cuda"), torch.rand(N, generator=gen, device="cuda")
        res = torch.randn(M, N, generator=gen, device="cuda")
        want = ops.gemm_int8(a[:, :K], sa, w[:, :K], sw, residual=res, out_dtype="fp32")
        p = _lib.GemmI8Args()
        p.M, p.N, p.K, p.out_dtype, p.lda, p.ldw, p.ldr, p.ldo = M, N, K, 0, a.stride(0), w.stride(0), N, N
        p.a, p.w, p.a_scale, p.w_scale, p.residual, p.out = (t.data_ptr() for t in (a, w, sa, sw, res, res))
        _lib.check(_lib.load().adcdiff_gemm_i8(C.byref(p), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(res, want)


@pytest.mark.parametrize("out", ["fp32", "bf16"])
@pytest.mark.parametrize("M, N, K, act", [(8200, 2051, 300, 0), (8200, 2051, 300, 1), (3000, 1003, 200, 1), (90, 77, 600, 0), (20, 301, 700, 1), (3, 5, 40, 0)])
def test_outputs_at_any_element(M, N, K, act, out):
    """odd widths, pitches and offsets of the residual and the output, in place (C ABI); nothing between the rows is written"""
    import ctypes as C
    from adcdiff import _lib
    gen = torch.Generator(device="cuda").manual_seed(8)
    a, w = _rows16(_codes(gen, M, K)), _rows16(_codes(gen, N, K))
    sa, sw = torch.rand(M, generator=gen, device="cuda"), torch.rand(N, generator=gen, device="cuda")
    pitch = N + 3
    held = torch.randn(M * pitch + 1, generator=gen, device="cuda").to(TYPES[out])
    before, rows = held.clone(), held[1:].view(M, pitch)[:, :N]
    want = ops.gemm_int8(a, sa, w, sw, residual=rows.contiguous(), act=act, out_dtype=out)
    p = _lib.GemmI8Args()
    p.M, p.N, p.K, p.act, p.out_dtype, p.lda, p.ldw, p.ldr, p.ldo = M, N, K, act, int(out == "bf16"), a.stride(0), w.stride(0), pitch, pitch
    p.a, p.w, p.a_scale, p.w_scale, p.residual, p.out = (t.data_ptr() for t in (a, w, sa, sw, rows, rows))
    _lib.check(_lib.load().adcdiff_gemm_i8(C.byref(p), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(rows, want)
    assert torch.equal(held[1:].view(M, pitch)[:, N:], before[1:].view(M, pitch)[:, N:]) and held[0] == before[0]


@pytest.mark.parametrize("M, N, K", [(1, 64, 1003), (50, 33, 77), (300, 1001, 515)])
def test_packed_codes(M, N, K):
    """codes without padding between rows, and at odd addresses"""
    _check(M, N, K, pad=False)
    gen = torch.Generator(device="cuda").manual_seed(1)
    held = _codes(gen, 1, M * K + 9)[0]
    a, w = held[5:5 + M * K].view(M, K), _codes(gen, N, K)
    one = torch.ones(max(M, N), device="cuda")
    y = ops.gemm_int8(a, one[:M], w, one[:N], out_dtype="fp32")
    assert torch.equal(y.double().cpu(), torch.mm(a.double().cpu(), w.double().cpu().t()).float().double())


def test_sums_are_exact_integers():
    gen = torch.Generator(device="cuda").manual_seed(2)
    for M, N, K in ((1, 2048, 2048), (32, 512, 1024), (512, 512, 1000), (4096, 2048, 512)):
        a, w = _codes(gen, M, K), _codes(gen, N, K)
        y = ops.gemm_int8(_rows16(a), torch.ones(M, device="cuda"), _rows16(w), torch.ones(N, device="cuda"), out_dtype="fp32")
        assert torch.equal(y.cpu(), torch.mm(a.double().cpu(), w.double().cpu().t()).float())      # int32 -> float32, one rounding
    for value in (-128, 127):
        a, w = torch.full((3, 131071), -128, dtype=torch.int8, device="cuda"), torch.full((20, 131071), value, dtype=torch.int8, device="cuda")
        y = ops.gemm_int8(_rows16(a), torch.ones(3, device="cuda"), _rows16(w), torch.ones(20, device="cuda"), out_dtype="fp32")
        assert bool((y == torch.tensor(float(-128 * value * 131071), dtype=torch.float64).float().cuda()).all())


def test_strided_output_rows_and_poison():
    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = _codes(gen, 40, 1024)
    a = wide[:, 256:256 + 500]                                     # other columns lie behind K
    w = _codes(gen, 70, 512)[:, :500]
    sa, sw = torch.rand(40, generator=gen, device="cuda"), torch.rand(70, generator=gen, device="cuda")
    sa[7] = float("nan")
    res = torch.randn(40, 100, generator=gen, device="cuda")[:, 3:73]
    y = ops.gemm_int8(a, sa, w, sw, residual=res, out_dtype="fp32")
    assert torch.isnan(y[7]).all()
    keep = [i for i in range(40) if i != 7]
    value, mag = ref.layer(a[keep], sa[keep], w, sw, None, res[keep], 0)
    ref.close(y[keep], value, mag, F, STEPS)
    assert ops.gemm_int8(a[:0], sa[:0], w, sw).shape == (0, 70)


def test_rows_past_32_bits():
    pitch = (1 << 31) + 64
    held = torch.empty(2 * pitch + 256, device="cuda", dtype=torch.int8)
    far = torch.as_strided(held, (3, 200), (pitch, 1))
    gen = torch.Generator(device="cuda").manual_seed(4)
    near, w = _codes(gen, 3, 200), _codes(gen, 90, 200)
    far.copy_(near)
    one = torch.ones(90, device="cuda")
    want = torch.mm(near.double().cpu(), w.double().cpu().t()).float()
    assert torch.equal(ops.gemm_int8(far, one[:3], _rows16(w), one, out_dtype="fp32").cpu(), want)
    assert torch.equal(ops.gemm_int8(_rows16(w), one, far, one[:3], out_dtype="fp32").cpu(), want.t())


@pytest.mark.parametrize("M", [1, 32, 700])
@pytest.mark.parametrize("dtype", [F, BF])
def test_layer_equals_its_two_halves(M, dtype):
    gen = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, 777, generator=gen, device="cuda").to(dtype)
    w, sw = ops.quantize_rows(torch.randn(300, 777, generator=gen, device="cuda"))
    b = torch.randn(300, generator=gen, device="cuda")
    q, s = ops.quantize_rows(x)
    y = ops.linear_int8(x, w, sw, bias=b, act=1, out_dtype="fp32")
    assert torch.equal(y, ops.gemm_int8(q, s, w, sw, bias=b, act=1, out_dtype="fp32"))
    value, mag = ref.layer(*ref.codes(x), w, sw, b, None, 1)
    ref.close(y, value, mag, F, STEPS + 2)       # the row's scale is itself rounded


def test_streams_and_graphs():
    """two graphs whose workspaces live side by side, replayed in turn with eager work between"""
    gen = torch.Generator(device="cuda").manual_seed(9)
    w, sw = ops.quantize_rows(torch.randn(512, 1000, generator=gen, device="cuda"))
    for M in (1, 32, 300):
        x = torch.randn(M, 1000, generator=gen, device="cuda")
        eager = ops.linear_int8(x, w, sw)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = ops.linear_int8(x, w, sw)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(eager, other)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = ops.linear_int8(x, w, sw)
            graphs.append((g, y))
        for _ in range(4):
            x.copy_(torch.randn(M, 1000, device="cuda"))
            eager = ops.linear_int8(x, w, sw)
            for g, y in graphs:
                g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(eager, y) for _, y in graphs)


def test_refusals():
    a, w = torch.zeros(4, 32, dtype=torch.int8, device="cuda"), torch.zeros(8, 32, dtype=torch.int8, device="cuda")
    sa, sw = torch.ones(4, device="cuda"), torch.ones(8, device="cuda")
    for call in (lambda: ops.gemm_int8(a, sa, w[:, :16], sw), lambda: ops.gemm_int8(a.float(), sa, w, sw), lambda: ops.gemm_int8(a, sa[:3], w, sw),
                 lambda: ops.gemm_int8(a, sa, w, sw.double()), lambda: ops.gemm_int8(a, sa, w, sw, bias=sa), lambda: ops.gemm_int8(a, sa, w, sw, residual=torch.zeros(4, 8, device="cuda")),
                 lambda: ops.gemm_int8(a, sa[:1].expand(4), w, sw), lambda: ops.gemm_int8(a[:, ::2], sa, w[:, ::2], sw), lambda: ops.quantize_rows(sa),
                 lambda: ops.quantize_rows(torch.zeros(3, 0, device="cuda")), lambda: ops.quantize_rows(torch.zeros(3, 8, device="cuda").half())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(adcdiff.AdcdiffError):
        ops.gemm_int8(a, sa, w, sw, act=3)


def test_gradients_are_refused():
    x = torch.randn(5, 40, device="cuda", requires_grad=True)
    w, sw = ops.quantize_rows(torch.randn(7, 40, device="cuda"))
    for y in (ops.linear_int8(x, w, sw), ops.quantize_rows(x)[1], ops.gemm_int8(w, sw, w, sw, bias=torch.zeros(7, device="cuda", requires_grad=True))):
        with pytest.raises(RuntimeError, match="no gradient"):
            y.sum().backward()
    assert torch.equal(ops.linear_int8(x, w, sw).detach(), ops.linear_int8(x.detach(), w, sw))


def test_operator_schemas():
    x = torch.randn(5, 40, device="cuda")
    q, s = ops.quantize_rows(x)
    utils = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.adcdiff.quantize_rows.default, (x,), test_utils=utils)
    torch.library.opcheck(torch.ops.adcdiff.gemm_int8.default, (q, s, q, s, None, None, 0, 1), test_utils=utils)
    torch.library.opcheck(torch.ops.adcdiff.linear_int8.default, (x, q, s, None, None, 1, 0), test_utils=utils)
