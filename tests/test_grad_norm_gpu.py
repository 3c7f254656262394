"""The gradient norm and clipping on the GPU against float64 and against torch.nn.utils.clip_grad_norm_'s rules.

Tolerances: the sum of squares is float64, so the norm is one float32 rounding (2^-24) from the exact one, plus the float64 sum's own
2^-53 per addition (nothing).  The factor takes three float32 roundings (sum, division, and the norm it starts from), the product one,
the store half a step of its type: 4 * 2^-24 + eps / 2 relative."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

adcdiff = pytest.importorskip("adcdiff")
from adcdiff import ops  # noqa: E402

BF, F = torch.bfloat16, torch.float32
U = 2.0 ** -24


def _tensors(sizes, dtype=F, scale=1.0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kinds = [F, BF] if dtype == "mixed" else [dtype]
    return [(torch.randn(n, generator=gen, device="cuda") * scale).to(kinds[i % len(kinds)]) for i, n in enumerate(sizes)]


def _norm64(ts):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


def _near(got, want):
    assert got.dtype == F and got.shape == ()
    assert abs(float(got) - want) <= U * want * 1.01, (float(got), want)


def _check_clip(before, after, out_types, max_norm, norm):
    factor = min(1.0, max_norm / (norm + 1e-6))
    for b, a, t in zip(before, after, out_types):
        assert a.dtype == t and a.shape == b.shape
        want = b.double() * factor
        assert bool(((a.double() - want).abs() <= (4 * U + torch.finfo(t).eps / 2 * 1.01) * want.abs() + 1e-38).all())


SIZES = [[1], [0], [5, 0, 3], [16384], [16385, 1, 16383], [7, 8, 9, 1023, 1025, 100003], [1 << 20, 3], list(range(1, 260)), [4097] * 121]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%d" % (len(s), max(s)))
@pytest.mark.parametrize("dtype", [F, BF, "mixed"])
def test_norm_and_clip(sizes, dtype):
    ts = _tensors(sizes, dtype)
    want = _norm64(ts)
    _near(ops.grad_norm(ts), want)
    assert float(ops.grad_norm(ts, norm_type=float("inf"))) == max([float(t.abs().max()) for t in ts if t.numel()], default=0.0)
    for max_norm in (0.0, 0.37, want + 1.0, float("inf")):
        got = [t.clone() for t in ts]
        _near(ops.clip_grad_norm_(got, max_norm), want)
        _check_clip(ts, got, [t.dtype for t in ts], max_norm, want)
    for kinds in ([F], [BF], [BF, F]):
        out = [torch.full(t.shape, 9.0, device="cuda", dtype=kinds[i % len(kinds)]) for i, t in enumerate(ts)]
        keep = [t.clone() for t in ts]
        _near(ops.clip_grad_norm_(ts, 0.37, out=out), want)
        _check_clip(ts, out, [o.dtype for o in out], 0.37, want)
        assert all(torch.equal(a, b) for a, b in zip(ts, keep))


def test_norm_type_inf_clips():
    ts = _tensors([1000, 33])
    top = max(float(t.abs().max()) for t in ts)
    got = [t.clone() for t in ts]
    assert float(ops.clip_grad_norm_(got, 0.5, norm_type="inf")) == top
    _check_clip(ts, got, [F, F], 0.5, top)


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5, 7])
def test_views_at_any_element(dtype, offset):
    """views into an arena, at every alignment of an element; what lies between them stays"""
    arena = torch.randn(60000, device="cuda").to(dtype)
    before = arena.clone()
    spans = [(offset, 17 + offset), (64 + offset, 20011), (20012 + offset, 40000), (40001, 40002), (40008 + offset, 59990)]
    views = [arena[a:b] for a, b in spans]
    want = _norm64(views)
    _near(ops.clip_grad_norm_(views, 1.0), want)
    _check_clip([before[a:b] for a, b in spans], views, [dtype] * len(spans), 1.0, want)
    inside = torch.zeros(60000, dtype=torch.bool, device="cuda")
    for a, b in spans:
        inside[a:b] = True
    assert torch.equal(arena[~inside], before[~inside])


def test_range_of_float32():
    """squares beyond float32's range in either direction"""
    for scale in (1e30, 1e-30, 1e-42, 3e38):
        ts = [torch.full((1000,), scale, device="cuda"), torch.full((5,), -scale / 2, device="cuda")]
        want = _norm64(ts)
        got = ops.grad_norm(ts)
        if want > 3.4e38:
            assert math.isinf(float(got))
        else:
            assert abs(float(got) - want) <= U * want + 1e-45


def test_not_finite():
    for bad in (float("nan"), float("inf"), -float("inf")):
        for dtype in (F, BF):
            ts = _tensors([100, 20000], dtype)
            ts[1][12345] = bad
            mine, theirs = [t.clone() for t in ts], [torch.nn.Parameter(t.clone()) for t in ts]
            for p, t in zip(theirs, ts):
                p.grad = t.clone()
            norm = ops.clip_grad_norm_(mine, 1.0)
            torch.nn.utils.clip_grad_norm_(theirs, 1.0)
            assert math.isnan(float(norm)) if math.isnan(bad) else math.isinf(float(norm))
            assert math.isnan(float(ops.grad_norm(ts, "inf"))) if math.isnan(bad) else math.isinf(float(ops.grad_norm(ts, "inf")))
            for a, p in zip(mine, theirs):
                assert torch.equal(torch.isnan(a), torch.isnan(p.grad)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(p.grad))
            keep = [t.clone() for t in ts]
            with pytest.raises(RuntimeError):
                ops.clip_grad_norm_(ts, 1.0, error_if_nonfinite=True)
            assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(ts, keep))


def test_layouts_and_refusals():
    t = torch.randn(40, 30, device="cuda")
    for view in (t.t(), t.view(8, 5, 30).permute(2, 0, 1), t[3]):
        _near(ops.grad_norm([view]), _norm64([view]))
    got = t.clone()
    ops.clip_grad_norm_([got.t()], 1.0)
    _check_clip([t], [got], [F], 1.0, _norm64([t]))
    _near(ops.grad_norm([t, t]), _norm64([t, t]))                 # read twice, counted twice
    for call in (lambda: ops.grad_norm([t[:, ::2]]), lambda: ops.grad_norm([t[:1].expand(4, 30)]), lambda: ops.grad_norm([t.half()]),
                 lambda: ops.clip_grad_norm_([t], 1.0, out=[torch.empty(30, 40, device="cuda")]),
                 lambda: ops.clip_grad_norm_([t.t()], 1.0, out=[torch.empty(30, 40, device="cuda")])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.clip_grad_norm_([t, t], 1.0), lambda: ops.clip_grad_norm_([t, t[2:4]], 1.0), lambda: ops.grad_norm([t, t.cpu()]),
                 lambda: ops.clip_grad_norm_([t[1:]], 1.0, out=[t[:-1]])):
        keep = t.clone()
        with pytest.raises(adcdiff.AdcdiffError):
            call()
        assert torch.equal(t, keep)


def test_versions_move():
    t, o = torch.randn(10, device="cuda"), torch.empty(10, device="cuda")
    a, b = t._version, o._version
    ops.clip_grad_norm_([t], 1.0, out=[o])
    assert t._version == a and o._version > b
    ops.clip_grad_norm_([t], 1.0)
    assert t._version > a
    ops.grad_norm([t])


def test_parameters_of_several_groups():
    """optim.clip_grad_norm_: torch.nn.utils.clip_grad_norm_'s signature over parameters"""
    from adcdiff import optim
    mine = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in (100, 7, 5000)] + [torch.nn.Parameter(torch.zeros(3, device="cuda"))]
    for p in mine[:3]:
        p.grad = torch.randn_like(p)
    before = [p.grad.clone() for p in mine[:3]]
    norm = optim.clip_grad_norm_(mine, 1.0)
    _near(norm, _norm64(before))
    _check_clip(before, [p.grad for p in mine[:3]], [F] * 3, 1.0, _norm64(before))
    assert float(optim.clip_grad_norm_([mine[3]], 1.0)) == 0.0


def test_streams_graphs_and_bits():
    ts = _tensors([100000, 5, 4097], "mixed")
    first = ops.grad_norm(ts)
    assert all(float(ops.grad_norm(ts)) == float(first) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.grad_norm(ts)
    torch.cuda.current_stream().wait_stream(side)
    assert float(other) == float(first)
    outs = [[torch.empty(t.shape, device="cuda") for t in ts] for _ in range(2)]
    graphs = []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norm = ops.clip_grad_norm_(ts, 0.5, out=outs[k])
        graphs.append((g, norm))
    for turn in range(4):
        for t in ts:
            t.copy_(torch.randn(t.shape, device="cuda") * (turn + 1))
        eager = [torch.empty(t.shape, device="cuda") for t in ts]
        want = ops.clip_grad_norm_(ts, 0.5, out=eager)
        for (g, norm), out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert float(norm) == float(want) and all(torch.equal(a, b) for a, b in zip(eager, out))


def test_operator_schemas():
    ts = _tensors([100, 5])
    utils = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.adcdiff.grad_norm.default, (ts, 2), test_utils=utils)
    torch.library.opcheck(torch.ops.adcdiff.clip_grad_norm_.default, (ts, 1.0, 2), test_utils=utils)
    torch.library.opcheck(torch.ops.adcdiff.clip_grad_norm_out.default, (ts, 1.0, 2, [torch.empty_like(t) for t in ts]), test_utils=utils)
