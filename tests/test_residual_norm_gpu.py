"""Gated residual norms on the GPU against the float64 form, forward and backward (tolerances: tests/block_reference.py)."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

adcdiff = pytest.importorskip("adcdiff")
from adcdiff import ops  # noqa: E402
import block_reference as ref  # noqa: E402

BF, F = torch.bfloat16, torch.float32
NAMES = ("h", "x", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")


def _inputs(M, D, T, R, GT, gates, post, pre, weights=True, seed=0, pitch=0, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 7919 * M + D)

    def rows(n, dtype, scale=1.0, shift=0.0):
        held = torch.full((n * (D + pitch) + offset + 8,), float("nan"), device="cuda", dtype=dtype)
        t = held[offset:offset + n * (D + pitch)].view(n, D + pitch)[:, :D]
        t.copy_(torch.randn(n, D, generator=gen, device="cuda") * scale + shift)
        return t

    s = {"h": rows(M, T, 1.5, 0.3), "x": rows(M, R, 2.0, -0.5), "gate": rows(gates, GT, 0.5, 0.2) if gates else None}
    for side, kind in (("post", post), ("pre", pre)):
        s[side + "_weight"] = 1.0 + 0.3 * torch.randn(D, generator=gen, device="cuda") if kind and weights else None
        s[side + "_bias"] = 0.2 * torch.randn(D, generator=gen, device="cuda") if kind and weights else None
    s["d_x"], s["d_y"] = rows(M, R), rows(M, T) if pre else None
    return s


def _check(s, post, pre, scale, eps=1e-6, steps=ref.STEPS, h=True):
    leaves = {k: s[k].detach() for k in NAMES if s[k] is not None and (h or k != "h")}
    for t in leaves.values():
        t.requires_grad_(True)
    get = leaves.get
    if h:
        xn, y = ops.residual_norm(get("h"), get("x"), gate=get("gate"), post_norm=post, post_weight=get("post_weight"), post_bias=get("post_bias"),
                                  pre_norm=pre, pre_weight=get("pre_weight"), pre_bias=get("pre_bias"), residual_scale=scale, eps=eps)
        outs, grads = [xn] + ([y] if pre else []), [s["d_x"]] + ([s["d_y"]] if pre else [])
    else:
        xn, y = None, ops.row_norm(get("x"), pre, get("pre_weight"), get("pre_bias"), eps)
        outs, grads = [y], [s["d_y"]]
    want = ref.residual_norm(s["h"].detach() if h else None, s["x"].detach(), s["gate"].detach() if h and s["gate"] is not None else None, post,
                             get("post_weight"), get("post_bias"), pre, get("pre_weight"), get("pre_bias"), scale, eps, s["d_x"] if h else None, s["d_y"])
    want = {k: (v.detach(), m.detach()) for k, (v, m) in want.items()}
    if h:
        ref.close(xn.detach(), *want["x_new"], s["x"].dtype)
    if pre:
        ref.close(y.detach(), *want["y"], outs[-1].dtype)
    got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads)))
    for k, g in got.items():
        value, mag = want[k]
        ref.close(g, value.view(g.shape), mag.expand_as(value).reshape(g.shape), s[k].dtype, steps + 64)
    for t in leaves.values():
        t.requires_grad_(False)
    return xn, y, got


WIDTHS = [1, 2, 7, 8, 16, 33, 128, 136, 512, 520, 777, 1024, 1032, 2048, 2049, 4096, 4100, 8184, 8192]


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("T, R", [(BF, BF), (BF, F), (F, F), (F, BF)])
def test_widths_and_types(D, T, R):
    for (post, pre), gates in zip((("rms", "rms"), ("layer", "layer")), (1, 9)):
        _check(_inputs(9, D, T, R, T, gates, post, pre), post, pre, 0.75, eps=1e-3)


@pytest.mark.parametrize("D", [3, 9, 15, 63, 127, 129, 255, 257, 511, 513, 517, 519, 521, 1025, 1535, 1537, 2051, 2561, 4095, 4097, 4103, 6143, 6145, 8191])
@pytest.mark.parametrize("T, R", [(BF, BF), (F, F)])
def test_last_columns(D, T, R):
    """rows whose last thread has fewer than eight columns of its own, behind a wave's end among them"""
    _check(_inputs(37, D, T, R, T, 37, "layer", "rms", pitch=1), "layer", "rms", 0.5)


@pytest.mark.parametrize("post, pre", list(itertools.product((None, "rms", "layer"), repeat=2)))
@pytest.mark.parametrize("gates", [0, 1, 6, 12])
def test_every_combination_of_parts(post, pre, gates):
    for weights in (True, False):
        _check(_inputs(12, 264, BF, F, F, gates, post, pre, weights), post, pre, 1.0)


@pytest.mark.parametrize("M, gates", [(1, 1), (2, 1), (3, 3), (64, 2), (1000, 1), (1000, 8), (1000, 500), (4099, 1), (5000, 1000), (20000, 4), (20000, 20000)])
@pytest.mark.parametrize("D", [64, 300, 1536])
def test_row_counts_and_groups(M, gates, D):
    """chunks that end inside a group, several chunks to a gate row, several gate rows to a workgroup; column sums over many rows
    add one rounding for each row that a thread adds up"""
    _check(_inputs(M, D, BF, F, BF, gates, "rms", "layer"), "rms", "layer", 0.5, steps=ref.STEPS + M // 64)


@pytest.mark.parametrize("pitch, offset", [(0, 1), (1, 0), (3, 5), (8, 0), (8, 8), (24, 4)])
@pytest.mark.parametrize("T, R", [(BF, BF), (F, F)])
def test_pitches_and_alignments(pitch, offset, T, R):
    for D in (96, 515, 2056):
        _check(_inputs(5, D, T, R, T, 5, "layer", "rms", pitch=pitch, offset=offset), "layer", "rms", 1.0)


@pytest.mark.parametrize("D", [5, 128, 1000, 5000])
@pytest.mark.parametrize("T", [BF, F])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_row_norm(D, T, kind):
    _check(_inputs(33, D, T, T, T, 0, None, kind), None, kind, 1.0, h=False)


def test_no_rows():
    s = _inputs(0, 64, BF, F, F, 0, "rms", "rms")
    gate = torch.randn(3, 64, device="cuda", requires_grad=True)
    w = s["pre_weight"].requires_grad_(True)
    s["h"].requires_grad_(True)
    xn, y = ops.residual_norm(s["h"], s["x"], gate=gate, post_norm="rms", pre_norm="rms", pre_weight=w)
    assert xn.shape == y.shape == (0, 64) and xn.dtype == F and y.dtype == BF
    g = torch.autograd.grad((xn, y), (s["h"], gate, w), (torch.zeros_like(xn), torch.zeros_like(y)))
    assert g[0].shape == (0, 64) and not g[1].any() and not g[2].any()
    assert ops.row_norm(s["x"]).shape == (0, 64)


def test_zero_rows_and_bad_rows_stay_by_themselves():
    s = _inputs(7, 264, F, F, F, 1, "rms", "layer")
    s["h"][1], s["x"][1] = 0.0, 0.0
    clean = ops.residual_norm(s["h"], s["x"], gate=s["gate"], post_norm="rms", pre_norm="layer")
    assert not clean[0][1].any() and not clean[1][1].any()          # 0 / sqrt(eps)
    for bad in (float("nan"), float("inf"), -float("inf")):
        h = s["h"].clone()
        h[3, 17] = bad
        xn, y = ops.residual_norm(h, s["x"], gate=s["gate"], post_norm="rms", pre_norm="layer")
        keep = [0, 1, 2, 4, 5, 6]
        assert torch.equal(xn[keep], clean[0][keep]) and torch.equal(y[keep], clean[1][keep])
        assert torch.isnan(y[3]).all()


def test_large_values_do_not_lose_the_variance():
    """a mean 4096 times the deviation: the centred sum keeps the variance (a difference of squares in float32 would lose it)"""
    x = 4096.0 + torch.randn(6, 1000, device="cuda")
    y = ops.row_norm(x, "layer")
    value, _, inv, mag = ref.norm(x, "layer", None, None, 1e-6)
    ref.close(y, value, mag, F)


def test_expanded_and_single_gates_are_the_same():
    s = _inputs(12, 264, BF, F, F, 1, "rms", "rms")
    a = ops.residual_norm(s["h"], s["x"], gate=s["gate"], post_norm="rms", pre_norm="rms")
    for gate in (s["gate"][0], s["gate"].expand(4, 264), s["gate"].expand(12, 264), s["gate"].repeat(12, 1)):
        b = ops.residual_norm(s["h"], s["x"], gate=gate, post_norm="rms", pre_norm="rms")
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    leaf = s["gate"][0].clone().requires_grad_(True)
    xn, _ = ops.residual_norm(s["h"], s["x"], gate=leaf.expand(4, 264), post_norm="rms", pre_norm="rms")
    g, = torch.autograd.grad(xn.sum(), leaf)       # the incoming gradient is one expanded number
    want = ref.residual_norm(s["h"], s["x"], s["gate"], "rms", None, None, None, None, None, 1.0, 1e-6, torch.ones_like(s["x"]))["gate"]
    ref.close(g, want[0][0], want[1][0], F, ref.STEPS + 64)


def test_partial_gradients():
    """each gradient alone, and with one incoming gradient missing, equals the one from the full backward pass"""
    s = _inputs(70, 520, BF, F, F, 7, "rms", "layer")
    xn, y, stats = torch.ops.adcdiff.residual_norm(*[s[k] for k in NAMES], 1, 2, 0.5, 1e-6, True, True)

    def back(d_x, d_y, need):
        return torch.ops.adcdiff.residual_norm_backward(*[s[k] for k in NAMES], stats, d_x, d_y, 1, 2, 0.5, 1e-6, need)
    full = back(s["d_x"], s["d_y"], [True] * 7)
    for i in range(7):
        if i == 2:      # the gate's gradient decides how rows are cut: the sums of the others then differ in order
            continue
        alone = back(s["d_x"], s["d_y"], [j in (i, 2) for j in range(7)])
        assert torch.equal(alone[0 if i < 2 else 1], full[i])
    zero = torch.zeros_like
    for a, b in ((back(None, s["d_y"], [True] * 7), back(zero(s["d_x"]), s["d_y"], [True] * 7)),
                 (back(s["d_x"], None, [True] * 7), back(s["d_x"], zero(s["d_y"]), [True] * 7))):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gradient_against_differences():
    """central differences of the float64 form along random directions (step 1e-5: their own error is below 1e-8 of the magnitudes)"""
    s = _inputs(40, 136, F, F, F, 5, "layer", "rms")
    _, _, got = _check(s, "layer", "rms", 0.7, eps=1e-3)

    def loss(**over):
        t = {k: s[k].double() for k in NAMES}
        t.update(over)
        out = ref.residual_norm(t["h"], t["x"], t["gate"], "layer", t["post_weight"], t["post_bias"], "rms", t["pre_weight"], t["pre_bias"], 0.7, 1e-3)
        return float((out["x_new"][0] * s["d_x"].double()).sum() + (out["y"][0] * s["d_y"].double()).sum())
    gen = torch.Generator(device="cuda").manual_seed(5)
    for k in NAMES:
        d = torch.randn(s[k].shape, generator=gen, device="cuda", dtype=torch.float64)
        diff = (loss(**{k: s[k].double() + 1e-5 * d}) - loss(**{k: s[k].double() - 1e-5 * d})) / 2e-5
        mine, mag = float((got[k].double() * d).sum()), float((got[k].double().abs() * d.abs()).sum())
        assert abs(mine - diff) <= (ref.STEPS * ref.U32 + 1e-6) * mag, k


def test_same_bits_every_run():
    s = _inputs(3001, 776, BF, BF, BF, 1, "rms", "rms")
    args = [s[k] for k in NAMES]
    first = None
    for _ in range(3):
        outs = torch.ops.adcdiff.residual_norm(*args, 1, 1, 1.0, 1e-6, True, True)
        outs = outs + torch.ops.adcdiff.residual_norm_backward(*args, outs[2], s["d_x"], s["d_y"], 1, 1, 1.0, 1e-6, [True] * 7)
        first = first or outs
        assert all(torch.equal(a, b) for a, b in zip(first, outs))


def test_offsets_past_32_bits():
    """rows more than 2^31 elements apart"""
    pitch = (1 << 30) + 40
    held = torch.empty(2 * pitch + 256, device="cuda", dtype=BF)
    far = torch.as_strided(held, (3, 256), (pitch, 1))
    near = torch.randn(3, 256, device="cuda").to(BF)
    far.copy_(near)
    a = ops.residual_norm(far, far, post_norm="rms", pre_norm="layer")
    b = ops.residual_norm(near, near, post_norm="rms", pre_norm="layer")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    nothing = 7 * [None]
    stats = torch.ops.adcdiff.residual_norm(near, near, *nothing[:5], 1, 2, 1.0, 1e-6, True, True)[2]
    need = [True, True] + 5 * [False]
    p = torch.ops.adcdiff.residual_norm_backward(far, far, *nothing[:5], stats, far, far, 1, 2, 1.0, 1e-6, need)
    q = torch.ops.adcdiff.residual_norm_backward(near, near, *nothing[:5], stats, near, near, 1, 2, 1.0, 1e-6, need)
    assert torch.equal(p[0], q[0]) and torch.equal(p[1], q[1])


@pytest.mark.parametrize("D", [3, 8, 9, 96, 513, 777, 1024, 4097, 8191])
@pytest.mark.parametrize("T, R", [(BF, F), (F, BF)])
def test_output_rows_with_gaps(D, T, R):
    """x_new and y at an odd pitch and offset (C ABI): the same values, and nothing between the rows is written"""
    import ctypes as C
    from adcdiff import _lib
    M, pitch = 61, D + 3
    s = _inputs(M, D, T, R, F, 1, "rms", "layer", pitch=1, offset=1)
    want = ops.residual_norm(s["h"], s["x"], gate=s["gate"], post_norm="rms", pre_norm="layer", residual_scale=0.5)
    held = [torch.full((M * pitch + 1,), 7.0, device="cuda", dtype=t) for t in (R, T)]
    xn, y = (t[1:].view(M, pitch) for t in held)
    a = _lib.ResidualNormArgs()
    a.M, a.D, a.dtype, a.stream_dtype, a.gate_dtype, a.post_norm, a.pre_norm, a.gate_rows = M, D, int(T == BF), int(R == BF), 0, 1, 2, 1
    a.h, a.x, a.x_new, a.y = s["h"].data_ptr(), s["x"].data_ptr(), xn.data_ptr(), y.data_ptr()
    a.gate, a.residual_scale, a.eps = s["gate"].data_ptr(), 0.5, 1e-6
    a.ldh, a.ldx, a.ldg, a.ldx_new, a.ldy = s["h"].stride(0), s["x"].stride(0), D, pitch, pitch
    _lib.check(_lib.load().adcdiff_residual_norm(C.byref(a), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(xn[:, :D], want[0]) and torch.equal(y[:, :D], want[1])
    assert bool((xn[:, D:] == 7.0).all()) and bool((y[:, D:] == 7.0).all()) and all(float(t[0]) == 7.0 for t in held)


@pytest.mark.parametrize("D", [5, 96, 513, 777, 1029, 2048, 4097, 8191, 8192])
def test_stream_in_place(D):
    """x_new over x and y over h (C ABI), with rows enough for every workgroup to take several"""
    import ctypes as C
    from adcdiff import _lib
    s = _inputs(9001, D, BF, F, F, 1, "rms", "layer")
    want = ops.residual_norm(s["h"], s["x"], gate=s["gate"], post_norm="rms", pre_norm="layer", residual_scale=0.5)
    a = _lib.ResidualNormArgs()
    a.M, a.D, a.dtype, a.stream_dtype, a.gate_dtype, a.post_norm, a.pre_norm, a.gate_rows = 9001, D, 1, 0, 0, 1, 2, 1
    a.h = a.y = s["h"].data_ptr()
    a.x = a.x_new = s["x"].data_ptr()
    a.gate, a.residual_scale, a.eps = s["gate"].data_ptr(), 0.5, 1e-6
    a.ldh = a.ldx = a.ldg = a.ldx_new = a.ldy = D
    _lib.check(_lib.load().adcdiff_residual_norm(C.byref(a), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(s["x"], want[0]) and torch.equal(s["h"], want[1])


def test_other_stream_and_graphs():
    s = _inputs(257, 1024, BF, F, F, 1, "rms", "rms")
    args = [s[k] for k in NAMES]

    def both():
        xn, y, stats = torch.ops.adcdiff.residual_norm(*args, 1, 1, 1.0, 1e-6, True, True)
        return [xn, y] + torch.ops.adcdiff.residual_norm_backward(*args, stats, s["d_x"], s["d_y"], 1, 1, 1.0, 1e-6, [True] * 7)
    eager = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = both()
        graphs.append((g, outs))
    for turn in range(4):
        s["h"].copy_(torch.randn(257, 1024, device="cuda"))
        s["d_y"].copy_(torch.randn(257, 1024, device="cuda"))
        eager = both()
        for g, outs in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(eager, outs)), turn


def test_autograd_function_under_capture():
    """forward and backward through autograd inside one graph, with no other graph of the leaves alive"""
    s = _inputs(64, 512, F, F, F, 1, "rms", "layer")
    leaves = [s[k].clone().requires_grad_(True) for k in ("h", "x", "gate")]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            xn, y = ops.residual_norm(leaves[0], leaves[1], gate=leaves[2], post_norm="rms", pre_norm="layer")
            torch.autograd.grad((xn, y), leaves, (s["d_x"], s["d_y"]))
        del xn, y
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        xn, y = ops.residual_norm(leaves[0], leaves[1], gate=leaves[2], post_norm="rms", pre_norm="layer")
        grads = torch.autograd.grad((xn, y), leaves, (s["d_x"], s["d_y"]))
    for _ in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn_like(leaves[0]))
        g.replay()
        torch.cuda.synchronize()
        fresh = [t.detach().clone().requires_grad_(True) for t in leaves]
        a, b = ops.residual_norm(fresh[0], fresh[1], gate=fresh[2], post_norm="rms", pre_norm="layer")
        assert torch.equal(a, xn) and torch.equal(b, y)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad((a, b), fresh, (s["d_x"], s["d_y"])), grads))


def test_differentiable_once():
    s = _inputs(6, 64, F, F, F, 2, "rms", "rms")
    h, x = s["h"].clone().requires_grad_(True), s["x"].clone().requires_grad_(True)
    xn, y = ops.residual_norm(h, x, gate=s["gate"], post_norm="rms", pre_norm="rms")
    g, = torch.autograd.grad(y.square().sum(), h, create_graph=True)
    plain, = torch.autograd.grad(ops.residual_norm(h, x, gate=s["gate"], post_norm="rms", pre_norm="rms")[1].square().sum(), h)
    assert torch.equal(g.detach(), plain)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


def test_outputs_without_gradient_inputs_have_none():
    s = _inputs(6, 64, F, F, F, 2, "rms", "rms")
    x = s["x"].clone().requires_grad_(True)
    assert not ops.residual_norm(s["h"], s["x"], pre_norm="rms")[1].requires_grad
    xn, y = ops.residual_norm(s["h"], x, pre_norm="rms")
    assert xn.requires_grad and y.requires_grad
    with torch.no_grad():
        assert not ops.residual_norm(s["h"], x, pre_norm="rms")[1].requires_grad
    g, = torch.autograd.grad(y.sum(), x)                 # x_new not used
    want = ref.residual_norm(s["h"], s["x"], None, None, None, None, "rms", None, None, 1.0, 1e-6, None, torch.ones_like(s["x"]))["x"]
    ref.close(g, *want, F, ref.STEPS + 64)
    x_changed = x.detach().clone().requires_grad_(True)
    y = ops.row_norm(x_changed)
    with torch.no_grad():
        x_changed.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_refusals():
    s = _inputs(6, 64, BF, F, F, 2, "rms", "rms")
    h, x = s["h"], s["x"]
    for call in (lambda: ops.residual_norm(h, x[:5]), lambda: ops.residual_norm(h[:, ::2], x[:, ::2]), lambda: ops.residual_norm(h.half(), x),
                 lambda: ops.residual_norm(h, x, gate=torch.zeros(4, 64, device="cuda")), lambda: ops.residual_norm(h, x, gate=torch.zeros(2, 32, device="cuda")),
                 lambda: ops.residual_norm(h, x, pre_weight=torch.ones(64, device="cuda")), lambda: ops.residual_norm(h, x, pre_norm="rms", pre_weight=torch.ones(63, device="cuda")),
                 lambda: ops.residual_norm(h, x, pre_norm="rms", pre_weight=torch.ones(64, device="cuda", dtype=BF)), lambda: ops.row_norm(x[0]),
                 lambda: ops.row_norm(x[:1].expand(6, 64))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.row_norm(torch.zeros(2, 8193, device="cuda")), lambda: ops.row_norm(x, eps=-1.0), lambda: ops.residual_norm(h, x.cpu())):
        with pytest.raises(adcdiff.AdcdiffError):
            call()


def test_operator_schemas():
    s = _inputs(6, 64, BF, F, F, 2, "rms", "rms")
    args = tuple(s[k] for k in NAMES)
    stats = torch.ops.adcdiff.residual_norm(*args, 1, 1, 1.0, 1e-6, True, True)[2]
    utils = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.adcdiff.residual_norm.default, args + (1, 1, 1.0, 1e-6, True, True), test_utils=utils)
    torch.library.opcheck(torch.ops.adcdiff.residual_norm_backward.default, args + (stats, s["d_x"], s["d_y"], 1, 1, 1.0, 1e-6, [True] * 7), test_utils=utils)
