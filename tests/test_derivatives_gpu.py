"""Derivatives that an operator does not have are refused on the GPU too (every operator and input: tests/test_derivatives_cpu.py)."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

adcdiff = pytest.importorskip("adcdiff")
from adcdiff import ops  # noqa: E402


def test_gradient_of_the_norm():
    p = torch.randn(4, 32, device="cuda", requires_grad=True)
    for kind in (2.0, "inf"):
        g, = torch.autograd.grad((p ** 3).sum(), p, create_graph=True)
        norm = ops.grad_norm([torch.zeros(3, device="cuda"), g], kind)
        assert torch.equal(norm.detach(), ops.grad_norm([g.detach()], kind))
        with pytest.raises(RuntimeError, match="grad_norm has no gradient"):
            (p.sum() + 0.1 * norm).backward()
    p.grad = torch.randn_like(p)
    before = p.grad.clone()
    assert not adcdiff.optim.clip_grad_norm_([p], 0.5).requires_grad      # .grad as an optimizer finds it: nothing changes
    assert bool((p.grad.norm() - 0.5).abs() < 1e-5) and not torch.equal(before, p.grad)


def test_tangents():
    x, w = torch.randn(4, 32, device="cuda"), torch.ones(32, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (ops.row_norm, ops.quantize_rows, lambda v: ops.groupnorm_silu(v, 4, w, w), lambda v: ops.clip_grad_norm_([v], 1.0)):
            with pytest.raises(NotImplementedError, match="forward"):
                call(dual)
        assert torch.equal(ops.row_norm(x), ops.row_norm(x.clone()))
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(ops.row_norm, (x,), (x,))
