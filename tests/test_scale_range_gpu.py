"""The 8-bit integer product over the whole range of its scales: the product of both scales and the sum has a value wherever it is a
float32, in whatever order it is formed.

Tolerance: the conversion of the sum, two products and the rounding of the output, 4 * 2^-24 relative, and for bfloat16 half a step more;
a result below the smallest normal number is off by one unit of 2^-149 (or of bfloat16's last bit there, 2^-133)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

adcdiff = pytest.importorskip("adcdiff")
from adcdiff import ops  # noqa: E402

U = 2.0 ** -24
EXPONENTS = (-126, -100, -64, -20, 0, 20, 64, 95, 96, 97, 110, 120, 126)


def _check(y, want):
    """finite and near where the exact value is a float32 (or bfloat16); beyond, infinity"""
    want = want.to(y.device)
    bf = y.dtype == torch.bfloat16
    rel = 4 * U + (torch.finfo(y.dtype).eps / 2 if bf else 0.0)
    top = torch.finfo(y.dtype).max
    inside = want.abs() <= top * (1 - rel)
    assert bool(inside.any()) and bool(torch.isfinite(y[inside]).all())
    err = (y.double() - want).abs()[inside]
    assert bool((err <= rel * want.abs()[inside] + 2.0 ** (-133 if bf else -149)).all()), float((err / want.abs()[inside].clamp(min=1e-44)).max())
    beyond = want.abs() > top * (1 + 2 * rel)
    assert bool(torch.isinf(y[beyond]).all()) and torch.equal(y[beyond] > 0, want[beyond] > 0)
    assert not y[want == 0].any()


# few rows, 64 x 64 and 128 x 128 tiles, 256 x 256 tiles
@pytest.mark.parametrize("out", ["fp32", "bf16"])
@pytest.mark.parametrize("M, N, K", [(13, 39, 2048), (100, 600, 700), (200, 1000, 700), (2080, 1300, 1024), (16640, 2080, 1024), (5300, 2056, 1024), (10384, 1027, 1643)])
def test_scales_of_any_magnitude(M, N, K, out):
    gen = torch.Generator(device="cuda").manual_seed(M + N)
    a = torch.randint(-128, 128, (M, K), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
    w = torch.randint(-128, 128, (N, K), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
    a[5] = 0                                                          # sums of zero under every scale
    e = torch.tensor(EXPONENTS, dtype=torch.float64, device="cuda")
    sa = ((1 + torch.rand(M, generator=gen, device="cuda").double()) * 2.0 ** e[torch.arange(M, device="cuda") % len(e)]).float()
    sw = ((1 + torch.rand(N, generator=gen, device="cuda").double()) * 2.0 ** e[torch.arange(N, device="cuda") // 3 % len(e)]).float()
    sums = torch.mm(a.double().cpu(), w.double().cpu().t()).cuda()
    y = ops.gemm_int8(a, sa, w, sw, out_dtype=out)
    _check(y, sums * sa.double()[:, None] * sw.double())


def test_layer_of_large_rows():
    """rows of 1e34 against weights of 1e-3: what a float32 product of the same rows gives without overflow"""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, wt = torch.rand(40, 2048, generator=gen, device="cuda") * 1e34, torch.rand(64, 2048, generator=gen, device="cuda") * 1e-3
    w, sw = ops.quantize_rows(wt)
    q, s = ops.quantize_rows(x)
    y = ops.linear_int8(x, w, sw, out_dtype="fp32")
    _check(y, torch.mm(q.double().cpu(), w.double().cpu().t()).cuda() * s.double()[:, None] * sw.double())
    assert bool(torch.isfinite(x @ wt.t()).all()) and bool((y / (x @ wt.t()) - 1).abs().max() < 0.05)
