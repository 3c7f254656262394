"""Derivatives on the GPU: what is refused (every operator and input: tests/test_derivatives_cpu.py), and what is a constant."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

adcdiff = pytest.importorskip("adcdiff")
from adcdiff import ops  # noqa: E402


def test_norms_of_parameters_in_a_compiled_step():
    """a step that returns the norm of its weights beside the loss: traced with the backward pass, and the gradient is the loss's alone"""
    p = torch.randn(40, 64, device="cuda", requires_grad=True)

    def step(x):
        return ops.row_norm(x * p).square().sum(), ops.grad_norm([p])
    x = torch.randn(40, 64, device="cuda")
    want, norm = step(x)
    got, traced = torch.compile(step, backend="aot_eager")(x)
    assert torch.equal(got, want) and torch.equal(traced, norm) and not traced.requires_grad
    assert torch.equal(torch.autograd.grad(got, p)[0], torch.autograd.grad(want, p)[0])
    assert norm.cpu().numpy() == ops.grad_norm([p.detach()]).cpu().numpy()


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
