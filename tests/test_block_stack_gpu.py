"""The operators together, as a user has them: a stack of conditioned residual blocks trained for a step (norms forward and backward,
products by torch, gradients clipped under one norm) and served in 8 bits (norms, row quantiser, integer product).  Every stage is
compared with the float64 form on the stage's own inputs, so no error is carried from one to the next."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

adcdiff = pytest.importorskip("adcdiff")
from adcdiff import ops, optim  # noqa: E402
import block_reference as ref  # noqa: E402

M, D, H, BLOCKS, GROUPS = 48, 160, 320, 3, 6


def _weights(seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return torch.nn.Parameter(torch.randn(*shape, generator=gen, device="cuda") * scale)
    blocks = [dict(pre=torch.nn.Parameter(torch.ones(D, device="cuda")), w1=rnd(H, D, scale=D ** -0.5), b1=rnd(H, scale=0.1), w2=rnd(D, H, scale=H ** -0.5),
                   post=rnd(D, scale=0.3), gate=rnd(GROUPS, D, scale=0.5)) for _ in range(BLOCKS)]
    return blocks, torch.randn(M, D, generator=gen, device="cuda"), torch.randn(M, D, generator=gen, device="cuda")


def _forward64(blocks, x):
    """the stack in plain float64 torch, differentiable"""
    def n(v, w):
        return v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * w
    y = n(x, blocks[0]["pre"])
    for i, b in enumerate(blocks):
        h = torch.nn.functional.silu(y @ b["w1"].t() + b["b1"]) @ b["w2"].t()
        x = 0.8 * x + b["gate"].repeat_interleave(M // GROUPS, dim=0) * n(h, b["post"])
        y = n(x, blocks[i + 1]["pre"]) if i + 1 < BLOCKS else x
    return y


def test_training_step():
    blocks, x, target = _weights()
    y, stream = ops.row_norm(x, "rms", blocks[0]["pre"]), x
    for i, b in enumerate(blocks):
        h = torch.nn.functional.silu(y @ b["w1"].t() + b["b1"]) @ b["w2"].t()
        last = i + 1 == BLOCKS
        stream, y = ops.residual_norm(h, stream, gate=b["gate"], post_norm="rms", post_weight=b["post"], pre_norm=None if last else "rms",
                                      pre_weight=None if last else blocks[i + 1]["pre"], residual_scale=0.8)
    ((stream - target) ** 2).mean().backward()
    leaves = [p for b in blocks for p in b.values()]
    plain = [{k: p.detach().double().requires_grad_(True) for k, p in b.items()} for b in blocks]
    out = _forward64(plain, x.double())
    ((out - target.double()) ** 2).mean().backward()
    wants = [p.grad for b in plain for p in b.values()]
    # float32 throughout: six products of at most 320 terms and four norms in a row, each within 200 roundings of its magnitude
    for p, w in zip(leaves, wants):
        assert float((p.grad.double() - w).norm()) <= 10 * ref.STEPS * ref.U32 * float(w.norm()) + 1e-12
    norm = math.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in leaves))
    before = [p.grad.clone() for p in leaves]
    got = optim.clip_grad_norm_(leaves, 0.5 * norm)
    assert abs(float(got) - norm) <= 1.01 * ref.U32 * norm
    for p, b in zip(leaves, before):
        assert bool(((p.grad - b * 0.5).abs() <= 8 * ref.U32 * b.abs() + 1e-6 / norm * b.abs()).all())
    opt = torch.optim.AdamW(leaves, lr=1e-3)
    opt.step()
    assert all(torch.isfinite(p).all() for p in leaves)


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
def test_serving_in_8_bits(T):
    blocks, x, _ = _weights(1)
    name = "bf16" if T == torch.bfloat16 else "fp32"
    with torch.no_grad():
        packed = [{"w1": ops.quantize_rows(b["w1"]), "w2": ops.quantize_rows(b["w2"])} for b in blocks]
        y, stream = ops.row_norm(x.to(T), "rms", blocks[0]["pre"]), x
        for i, (b, q) in enumerate(zip(blocks, packed)):
            last = i + 1 == BLOCKS
            t = ops.linear_int8(y, *q["w1"], bias=b["b1"], act=1, out_dtype=name)
            h = ops.linear_int8(t, *q["w2"], out_dtype=name)
            for got, inp, key, bias, act in ((t, y, "w1", b["b1"], 1), (h, t, "w2", None, 0)):
                value, mag = ref.layer(*ref.codes(inp), *q[key], bias, None, act)
                ref.close(got, value, mag, T, 12)
            want = ref.residual_norm(h, stream, b["gate"], "rms", b["post"], None, None if last else "rms", None if last else blocks[i + 1]["pre"], None, 0.8, 1e-6)
            stream, y = ops.residual_norm(h, stream, gate=b["gate"], post_norm="rms", post_weight=b["post"], pre_norm=None if last else "rms",
                                          pre_weight=None if last else blocks[i + 1]["pre"], residual_scale=0.8)
            ref.close(stream, *want["x_new"], torch.float32)
            if not last:
                ref.close(y, *want["y"], T)
    assert torch.isfinite(stream).all()
