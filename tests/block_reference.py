"""Plain float64 forms of the operators around a residual block, and the tolerances their float32 forms are held to.

Tolerances.  A value that is rounded once to a type t is off by at most half a step, eps(t) / 2 relative to it.  In front of that
rounding the kernels compute in float32 (half step 2^-24).  An element of a row passes through at most
  12 element-wise operations,  the four statistics / means it uses, each a sum of D products: D / (8 .. 1024 threads) sequential
  additions per thread (at most 32) and at most 10 in the tree over the threads, plus 5 operations to finish it,
so about 12 + 4 * 47 = 200 roundings, each relative to at most the largest intermediate magnitude S of that row, which the functions here
return beside the value (sums of absolute values, so cancellation is counted).  Errors of independent roundings add far slower than
their number; the bound used is 200 * 2^-24 * S, with nothing left out of S.  A sum over rows adds the rows' own bounds, plus one
rounding per addition (at most 64 sequential ones per thread and chunk) relative to the sum of magnitudes: (200 + 64) * 2^-24 * sum S."""
import torch

U32 = 2.0 ** -24
STEPS = 200


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, ref, scale, dtype, steps=STEPS):
    """Asserts |got - ref| <= half a step of the output's type + steps * 2^-24 * scale, element by element."""
    assert got.dtype == dtype and got.shape == ref.shape, (got.dtype, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    bound = half_step(dtype) * ref.abs() * (1 + 2 ** -7) + steps * U32 * scale + 1e-37
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0, "error of %.3g times the bound" % worst
    return worst


def norm(v, kind, weight, bias, eps):
    """(output, unit, 1 / deviation, magnitude of the output's intermediates per row) in float64"""
    mag = v.abs().amax(dim=1, keepdim=True)
    c = v - v.mean(dim=1, keepdim=True) if kind == "layer" else v
    inv = 1.0 / torch.sqrt((c * c).mean(dim=1, keepdim=True) + eps)
    unit = c * inv
    w = torch.ones(v.shape[1], dtype=torch.float64, device=v.device) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    return unit * w + b, unit, inv, mag * inv


def residual_norm(h, x, gate, post_norm, post_weight, post_bias, pre_norm, pre_weight, pre_bias, scale, eps, d_x=None, d_y=None):
    """x_new, y and, given incoming gradients, every gradient: a dict of (value, magnitude), all float64."""
    M, D = x.shape
    x = x.double()
    out = {}
    group = None
    if gate is not None:
        gate2 = gate.double().reshape(-1, D)
        group = torch.arange(M, device=x.device) // max(1, M // gate2.shape[0])
    if h is not None:
        h = h.double()
        u, u_mag = h, h.abs()
        if post_norm:
            u, u_unit, u_inv, m = norm(h, post_norm, post_weight, post_bias, eps)
            w = 1.0 if post_weight is None else post_weight.double().abs()
            u_mag = m * w + (0.0 if post_bias is None else post_bias.double().abs())
        g = 1.0 if gate is None else gate2[group]
        xn = scale * x + g * u
        xn_mag = abs(scale) * x.abs() + (1.0 if gate is None else g.abs()) * u_mag
    else:
        u, g, xn, xn_mag = None, 1.0, x, x.abs()
    out["x_new"] = (xn, xn_mag)
    if pre_norm:
        y, unit, inv, _ = norm(xn, pre_norm, pre_weight, pre_bias, eps)
        row_mag = xn_mag.amax(dim=1, keepdim=True) * inv            # magnitude of anything in the normalised row
        w = torch.ones(D, dtype=torch.float64, device=x.device) if pre_weight is None else pre_weight.double()
        out["y"] = (y, row_mag * w.abs() + (0.0 if pre_bias is None else pre_bias.double().abs()))
    if d_x is None and d_y is None:
        return out
    d = torch.zeros_like(x) if d_x is None else d_x.double()
    d_mag = d.abs().amax(dim=1, keepdim=True)
    if pre_norm:
        dy = torch.zeros_like(x) if d_y is None else d_y.double()
        gy = dy * w
        g_mag = gy.abs().amax(dim=1, keepdim=True)
        d = d + inv * (gy - (gy.mean(dim=1, keepdim=True) if pre_norm == "layer" else 0.0) - unit * (gy * unit).mean(dim=1, keepdim=True))
        unit_mag = torch.maximum(row_mag, unit.abs().amax(dim=1, keepdim=True))
        d_mag = d_mag + inv * g_mag * (2 + unit_mag * unit_mag)
        out["pre_weight"] = ((dy * unit).sum(dim=0), (dy.abs() * unit_mag).sum(dim=0))
        out["pre_bias"] = (dy.sum(dim=0), dy.abs().sum(dim=0))
    d_mag = d_mag.expand(M, D)
    out["x"] = (scale * d, abs(scale) * d_mag)
    if h is None:
        return out
    if gate is not None:
        G = gate2.shape[0]
        out["gate"] = ((d * u).view(G, -1, D).sum(dim=1), (d_mag * u_mag).view(G, -1, D).sum(dim=1))
    dh, dh_mag = d * g, d_mag * (1.0 if gate is None else g.abs().amax(dim=1, keepdim=True))
    if post_norm:
        out["post_weight"] = ((dh * u_unit).sum(dim=0), (dh_mag * m).sum(dim=0))
        out["post_bias"] = (dh.sum(dim=0), dh_mag.sum(dim=0))
        w = torch.ones(D, dtype=torch.float64, device=x.device) if post_weight is None else post_weight.double()
        gp = dh * w
        gp_mag = (dh_mag * w.abs()).amax(dim=1, keepdim=True)
        dh = u_inv * (gp - (gp.mean(dim=1, keepdim=True) if post_norm == "layer" else 0.0) - u_unit * (gp * u_unit).mean(dim=1, keepdim=True))
        dh_mag = u_inv * gp_mag * (2 + m * m)
    out["h"] = (dh, dh_mag.expand(M, D))
    return out


def codes(x):
    """(codes, scale) of rows in float64: half to even, zeros for a row of zeros, codes 0 and scale NaN for a row with NaN or infinity"""
    x = x.double()
    top = x.abs().amax(dim=1, keepdim=True)
    bad = ~torch.isfinite(x).all(dim=1, keepdim=True)
    q = torch.round(x * 127.0 / torch.where((top > 0) & ~bad, top, 1.0))
    q = torch.where(bad, 0.0, q)
    return q, torch.where(bad, float("nan"), top / 127.0)[:, 0]


def layer(a, a_scale, w, w_scale, bias, residual, act):
    """(value, magnitude) of the 8-bit integer layer from its codes"""
    v = torch.mm(a.double().cpu(), w.double().cpu().t()).to(a.device) * a_scale.double()[:, None] * w_scale.double()
    mag = v.abs()
    for t in (bias, residual):
        if t is not None:
            v, mag = v + t.double(), mag + t.double().abs()
    if act:
        v, mag = v * torch.sigmoid(v), mag * 1.2     # |d silu / d v| < 1.1
    return v, mag
