"""Derivatives that an operator does not have are refused, never left out: a result without a tangent counts as
constant.  On fake tensors: the refusals come before any kernel."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

import adcdiff
from adcdiff import ops


def _gpu(*shape, dtype=torch.float32):
    return torch.empty(*shape, device="cuda", dtype=dtype)


def _i8(rows):
    return _gpu(rows, 32, dtype=torch.int8), _gpu(rows)


def _backward(d_y):
    return torch.ops.adcdiff.residual_norm_backward(None, _gpu(4, 32), None, None, None, None, None, _gpu(4, 4), None, d_y, 0, 1, 1.0, 1e-6,
                                                    [False, True] + 5 * [False])


# one for each way a [4, 32] float32 tensor enters an operator
CALLS = {
    "row_norm": lambda d: ops.row_norm(d),
    "row_norm weight": lambda d: ops.row_norm(_gpu(4, 128), weight=d.reshape(128)),
    "residual_norm h": lambda d: ops.residual_norm(d, _gpu(4, 32)),
    "residual_norm x": lambda d: ops.residual_norm(_gpu(4, 32), d, pre_norm="rms"),
    "residual_norm gate": lambda d: ops.residual_norm(_gpu(4, 32), _gpu(4, 32), gate=d),
    "residual_norm bias": lambda d: ops.residual_norm(_gpu(4, 128), _gpu(4, 128), post_norm="layer", post_bias=d.reshape(128)),
    "residual_norm_backward": _backward,
    "quantize_rows": lambda d: ops.quantize_rows(d),
    "gemm_int8 residual": lambda d: ops.gemm_int8(*_i8(4), *_i8(32), residual=d, out_dtype="fp32"),
    "gemm_int8 scale": lambda d: ops.gemm_int8(*_i8(4), _gpu(128, 32, dtype=torch.int8), d.reshape(128)),
    "linear_int8": lambda d: ops.linear_int8(d, *_i8(7)),
    "linear_int8 bias": lambda d: ops.linear_int8(_gpu(4, 32), *_i8(128), bias=d.reshape(128)),
    "grad_norm": lambda d: ops.grad_norm([_gpu(3), d]),
    "clip_grad_norm_": lambda d: ops.clip_grad_norm_([_gpu(3), d], 1.0),
    "clip_grad_norm_ from": lambda d: ops.clip_grad_norm_([d], 1.0, out=[_gpu(4, 32)]),
    "clip_grad_norm_ into": lambda d: ops.clip_grad_norm_([_gpu(4, 32)], 1.0, out=[d]),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_forward_mode_is_refused(name):
    call = CALLS[name]
    with FakeTensorMode():
        call(_gpu(4, 32))
        with forward_ad.dual_level():
            call(_gpu(4, 32))
            dual = forward_ad.make_dual(_gpu(4, 32), _gpu(4, 32))
            with pytest.raises(NotImplementedError, match="forward"):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):     # forward mode goes on there
                call(dual)
            with forward_ad._set_fwd_grad_enabled(False):
                call(dual)
        with pytest.raises(NotImplementedError, match="forward"):
            torch.func.jvp(lambda v: (call(v), v)[1], (_gpu(4, 32),), (_gpu(4, 32),))


# functions of the sampling path, on the CPU: the refusal comes before the one of CPU tensors
PATH_CALLS = {
    "gemm a": lambda d: ops.gemm([d], torch.empty(16, 32)),
    "gemm w": lambda d: ops.gemm([torch.empty(4, 32)], d),
    "gemm residual": lambda d: ops.gemm([torch.empty(4, 8)], torch.empty(32, 8), residual=d),
    "groupnorm_silu x": lambda d: ops.groupnorm_silu(d, 4, torch.ones(32), torch.zeros(32)),
    "groupnorm_silu gamma": lambda d: ops.groupnorm_silu(torch.ones(4, 128), 4, d.reshape(128), torch.zeros(128)),
    "ddpm_step": lambda d: ops.ddpm_step(d, torch.empty(4, 32), (1.0, 0.1, 0.5, 0.2)),
    "ddim_step": lambda d: ops.ddim_step(torch.empty(4, 32), d, (1.0, 0.1, 0.5, 0.2, 0.1)),
    "q_sample": lambda d: ops.q_sample(d, torch.zeros(4, dtype=torch.int64), torch.ones(10), torch.ones(10)),
    "latent_summary": lambda d: ops.latent_summary(d),
    "model": lambda d: adcdiff.UNetModel(32, 32, 32, 10, strict_shapes=False)(d, torch.zeros(4, dtype=torch.int64)),
}


@pytest.mark.parametrize("name", list(PATH_CALLS))
def test_forward_mode_of_the_path_is_refused(name):
    call = PATH_CALLS[name]
    with forward_ad.dual_level():
        with pytest.raises(adcdiff.AdcdiffError):     # as without forward mode: no CPU path
            call(torch.zeros(4, 32))
        with pytest.raises(NotImplementedError, match="forward"):
            call(forward_ad.make_dual(torch.zeros(4, 32), torch.zeros(4, 32)))
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(call, (torch.zeros(4, 32),), (torch.zeros(4, 32),))


def test_norms_are_constants():
    """of tensors that require a gradient too, as the total norm of torch.nn.utils is; a compiled step may return them beside its loss"""
    with FakeTensorMode():
        p = _gpu(4, 32).requires_grad_()
        for call in (lambda: ops.grad_norm([_gpu(3), p * 2.0]), lambda: ops.grad_norm([p], "inf"), lambda: ops.clip_grad_norm_([p * 2.0], 1.0),
                     lambda: ops.clip_grad_norm_([p * 2.0], 1.0, out=[_gpu(4, 32)])):
            norm = call()
            assert norm.shape == () and norm.dtype == torch.float32 and not norm.requires_grad
