"""The operators around a denoiser's residual block, measured: the 8-bit integer layer that serves it, the norms before and after
it with its gate and residual scale (inference and training), and the global gradient norm with its clipping.

``run`` computes a case in its plain form (elementary torch operations in 32 bits) or, where ``own`` is true, through the
framework's entry points; ``exact`` computes it in 64 bits from the definitions.

The definitions:
  codes of a row      scale = max|x| / 127,  code = round_half_even(x * 127 / max|x|)
  8-bit integer layer y[m, n] = act(a_scale[m] * w_scale[n] * sum_k a[m, k] w[n, k] + bias[n] + residual[m, n]),  act: none or v * sigmoid(v)
  norm of a row       rms: v / sqrt(mean(v^2) + eps) * weight + bias;  layer: the same of v - mean(v)
  gated residual norm x' = residual_scale * x + gate * N_post(h),  y = N_pre(x');  row r reads gate row r // (rows / gate rows)
  clipping            norm = sqrt(sum over all tensors of g^2),  g * min(1, max_norm / (norm + 1e-6))
"""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
LARGEST_PRODUCT = 65536 * 2048 * 2048
LARGEST_ROWS = 65536 * 2048


def listed():
    return [
        # one request: one row through a square layer whose codes are ready; the weights' bytes and the launch are all there is
        {"name": "int8_product_one_row", "op": "product", "rows": 1, "out": 2048, "inner": 2048, "type": "bf16", "bias": True,
         "residual": False, "act": 0, "pitch16": True},
        # the generator's batch of 32 latents through the widest contraction of the denoiser (skip concatenation), from float32 rows
        {"name": "int8_layer_batch32", "op": "layer", "rows": 32, "out": 2048, "inner": 4096, "type": "fp32", "bias": True,
         "residual": False, "act": 0},
        # nothing divides anything: odd rows, outputs and inner length, codes packed without padding, float32 result
        {"name": "int8_product_ragged", "op": "product", "rows": 777, "out": 1000, "inner": 1003, "type": "fp32", "bias": True,
         "residual": True, "act": 0, "pitch16": False},
        # an ordinary layer of a training-sized batch, bf16 rows in, SiLU fused
        {"name": "int8_layer_batch4096", "op": "layer", "rows": 4096, "out": 2048, "inner": 2048, "type": "bf16", "bias": True,
         "residual": False, "act": 1},
        # the benchmark's sampling batch: one large product with bias and residual
        {"name": "int8_product_batch65536", "op": "product", "rows": 65536, "out": 2048, "inner": 2048, "type": "bf16", "bias": True,
         "residual": True, "act": 0, "pitch16": True},
        # sampling 32 latents: the seam between two blocks, one gate for all rows; latency
        {"name": "norm_batch32", "op": "norm", "train": False, "rows": 32, "width": 512, "type": "bf16", "stream": "fp32", "post": "rms",
         "pre": "rms", "gates": 1, "residual_scale": 1.0},
        # the benchmark's sampling batch, every row with a gate of its own (per-row timesteps)
        {"name": "norm_batch65536", "op": "norm", "train": False, "rows": 65536, "width": 2048, "type": "bf16", "stream": "bf16",
         "post": "rms", "pre": "rms", "gates": 65536, "residual_scale": 1.0},
        # a training step's seam, float32 with layer norms and one learned gate: both directions
        {"name": "norm_train_batch4096", "op": "norm", "train": True, "rows": 4096, "width": 1024, "type": "fp32", "stream": "fp32",
         "post": "layer", "pre": "layer", "gates": 1, "residual_scale": 0.70710678},
        # bf16 training of many rows in 64 groups that share a gate (one per molecule, several rows each), float32 residual stream
        {"name": "norm_train_batch32768", "op": "norm", "train": True, "rows": 32768, "width": 2048, "type": "bf16", "stream": "fp32",
         "post": "rms", "pre": "rms", "gates": 64, "residual_scale": 1.0},
        # odd everything, a norm before the next block only
        {"name": "norm_train_ragged", "op": "norm", "train": True, "rows": 1003, "width": 777, "type": "bf16", "stream": "bf16",
         "post": "", "pre": "layer", "gates": 17, "residual_scale": 0.5},
        # gradients of a small head: six short tensors, all launch
        {"name": "grad_norm_small", "op": "grad_norm", "clip": False, "blocks": 1, "width": 64, "type": "fp32", "max_norm": 1.0},
        # the denoiser's 44 million gradients in 70 tensors, clipped into the optimizer's arena
        {"name": "grad_clip_denoiser", "op": "grad_norm", "clip": True, "blocks": 14, "width": 1024, "type": "fp32", "max_norm": 1.0},
    ]


def _spread(rng, low, high):
    """a whole number, even over the logarithm of the range"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["product", "layer", "norm", "norm", "grad_norm"])
    kind = rng.choice(["bf16", "fp32"])
    if op in ("product", "layer"):
        rows, out, inner = _spread(rng, 1, 65536), _spread(rng, 32, 4096), _spread(rng, 32, 8192)
        rows = max(1, min(rows, LARGEST_PRODUCT // (out * inner), LARGEST_ROWS // max(out, inner)))
        case = {"op": op, "rows": rows, "out": out, "inner": inner, "type": kind, "bias": rng.random() < 0.7,
                "residual": op == "product" and rng.random() < 0.5, "act": rng.randrange(2)}
        if op == "product":
            case["pitch16"] = rng.random() < 0.8
        return case
    if op == "norm":
        width = _spread(rng, 16, 8192)
        width += (-width) % rng.choice([1, 8, 64])
        rows = max(1, min(_spread(rng, 1, 65536), LARGEST_ROWS // (2 * width)))
        groups = rng.choice([1, rows, 0])
        if groups == 0:  # several rows to a gate
            share = min(rows, _spread(rng, 2, 512))
            groups = max(1, rows // share)
            rows = groups * share
        return {"op": "norm", "train": rng.random() < 0.6, "rows": rows, "width": width, "type": kind, "stream": rng.choice([kind, "fp32"]),
                "post": rng.choice(["rms", "layer", ""]), "pre": rng.choice(["rms", "layer"]), "gates": groups,
                "residual_scale": rng.choice([1.0, 0.5, 0.70710678])}
    width = _spread(rng, 16, 2048)
    return {"op": "grad_norm", "clip": rng.random() < 0.5, "blocks": max(1, min(_spread(rng, 1, 40), 44_000_000 // (3 * width * width))),
            "width": width, "type": kind, "max_norm": rng.choice([0.5, 1.0, 1e4])}


# ------------------------------------------------------------------------------------------------------------- inputs
def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * scale


def _rows(gen, rows, width):
    """activations: normal with a spread of row magnitudes and a few strong channels"""
    x = _normal(gen, rows, width)
    x *= torch.exp(0.5 * _normal(gen, rows, 1))
    return x * (1.0 + 4.0 * (torch.rand(width, generator=gen, device="cuda") < 0.01))


def _stored(codes, pitch16):
    """codes whose rows start on 16-byte boundaries (as the framework's row quantiser leaves them) or directly behind each other"""
    rows, width = codes.shape
    if not pitch16:
        return codes
    held = torch.zeros(rows, (width + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    held[:, :width] = codes
    return held[:, :width]


def _quantise(x):
    top = x.double().abs().amax(dim=1)
    codes = torch.round(x.double() * 127.0 / torch.where(top > 0, top, 1.0)[:, None])
    return codes.to(torch.int8), (top / 127.0).float()


def _gradient_shapes(case):
    w = case["width"]
    return [shape for _ in range(case["blocks"]) for shape in ((w, w), (w,), (w, 2 * w), (w,), (w,))]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]
    s = {"case": case}
    if case["op"] in ("product", "layer"):
        M, N, K = case["rows"], case["out"], case["inner"]
        w, w_scale = _quantise(_normal(gen, N, K, scale=K ** -0.5))
        s.update(w=_stored(w, case.get("pitch16", True)), w_scale=w_scale)
        x = _rows(gen, M, K)
        if case["op"] == "product":
            a, s["a_scale"] = _quantise(x)
            s["a"] = _stored(a, case["pitch16"])
        else:
            s["x"] = x.to(kind)
        s["bias"] = _normal(gen, N, scale=0.1) if case["bias"] else None
        s["residual"] = _normal(gen, M, N).to(kind) if case["residual"] else None
        return s
    if case["op"] == "norm":
        M, D, train = case["rows"], case["width"], case["train"]
        stream = TYPES[case["stream"]]
        s["h"] = _rows(gen, M, D).to(kind)
        s["x"] = (2.0 * _rows(gen, M, D)).to(stream)
        s["gate"] = (0.3 + 0.3 * _normal(gen, case["gates"], D)).to(kind)
        for side in ("post", "pre"):
            s[side + "_weight"] = 1.0 + 0.1 * _normal(gen, D) if case[side] else None
            s[side + "_bias"] = 0.1 * _normal(gen, D) if case[side] == "layer" else None
        s["leaves"] = [k for k in ("h", "x", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if s[k] is not None]
        if train:
            s["grad_x"] = _normal(gen, M, D, scale=1.0 / M).to(stream)
            s["grad_y"] = _normal(gen, M, D, scale=1.0 / M).to(kind)
            for k in s["leaves"]:
                s[k].requires_grad_(True)
        return s
    shapes = _gradient_shapes(case)
    s["grads"] = []
    for shape in shapes:
        s["grads"].append((_normal(gen, *shape) * (0.02 * math.exp(-0.5 * len(s["grads"]) / len(shapes)))).to(kind))
    if case["clip"]:  # the optimizer's float32 gradient arena and its views
        s["arena"] = torch.empty(sum(g.numel() for g in s["grads"]), device="cuda")
        s["views"], at = [], 0
        for g in s["grads"]:
            s["views"].append(s["arena"][at:at + g.numel()].view(g.shape))
            at += g.numel()
    return s


# ------------------------------------------------------------------------------------------------------------- plain forms
def _plain_product(a, a_scale, s):
    v = (a.float() @ s["w"].float().t()) * a_scale[:, None] * s["w_scale"]
    if s["bias"] is not None:
        v = v + s["bias"]
    if s["residual"] is not None:
        v = v + s["residual"].float()
    if s["case"]["act"]:
        v = v / (1.0 + torch.exp(-v))
    return v.to(TYPES[s["case"]["type"]])


def _plain_norm(v, kind, weight, bias):
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS) * weight
    return y if bias is None else y + bias


def _plain_residual_norm(s):
    c = s["case"]
    u = s["h"].float()
    if c["post"]:
        u = _plain_norm(u, c["post"], s["post_weight"], s["post_bias"])
    share = c["rows"] // c["gates"]
    gated = (u.view(c["gates"], share, -1) * s["gate"].float()[:, None, :]).view(c["rows"], -1)
    x = c["residual_scale"] * s["x"].float() + gated
    return x.to(s["x"].dtype), _plain_norm(x, c["pre"], s["pre_weight"], s["pre_bias"]).to(s["h"].dtype)


def _plain_clip(s):
    norm = torch.sqrt(torch.stack([g.float().square().sum() for g in s["grads"]]).sum())
    if not s["case"]["clip"]:
        return norm
    factor = torch.clamp(s["case"]["max_norm"] / (norm + 1e-6), max=1.0)
    torch.cat([(g.float() * factor).reshape(-1) for g in s["grads"]], out=s["arena"])
    return {"norm": norm, "clipped": s["arena"]}


# ------------------------------------------------------------------------------------------------------------- own
def _own_product(s):
    from adcdiff import ops
    c = s["case"]
    if c["op"] == "layer":
        return ops.linear_int8(s["x"], s["w"], s["w_scale"], bias=s["bias"], act=c["act"], out_dtype=c["type"])
    return ops.gemm_int8(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"], residual=s["residual"], act=c["act"], out_dtype=c["type"])


def _own_residual_norm(s):
    from adcdiff import ops
    c = s["case"]
    return ops.residual_norm(s["h"], s["x"], gate=s["gate"], post_norm=c["post"] or None, post_weight=s["post_weight"],
                             post_bias=s["post_bias"], pre_norm=c["pre"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"],
                             residual_scale=c["residual_scale"], eps=EPS)


def _own_clip(s):
    from adcdiff import ops
    if not s["case"]["clip"]:
        return ops.grad_norm(s["grads"])
    norm = ops.clip_grad_norm_(s["grads"], s["case"]["max_norm"], out=s["views"])
    return {"norm": norm, "clipped": s["arena"]}


def run(s):
    c = s["case"]
    if c["op"] in ("product", "layer"):
        if own:
            return _own_product(s)
        a, a_scale = _quantise(s["x"]) if c["op"] == "layer" else (s["a"], s["a_scale"])
        return _plain_product(a, a_scale, s)
    if c["op"] == "norm":
        x, y = _own_residual_norm(s) if own else _plain_residual_norm(s)
        if not c["train"]:
            return {"x": x, "y": y}
        grads = torch.autograd.grad((x, y), [s[k] for k in s["leaves"]], (s["grad_x"], s["grad_y"]))
        return {"x": x.detach(), "y": y.detach(), "grads": dict(zip(s["leaves"], grads))}
    return _own_clip(s) if own else _plain_clip(s)


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] in ("product", "layer"):
        M, N, K = case["rows"], case["out"], case["inner"]
        rows = M * K * size if case["op"] == "layer" else M * (K + 4)
        nbytes = rows + N * (K + 4) + M * N * size * (2 if case["residual"] else 1) + (4 * N if case["bias"] else 0)
        return {"bytes": nbytes, "flops": 2.0 * M * N * K}
    if case["op"] == "norm":
        M, D, stream = case["rows"], case["width"], 2 if case["stream"] == "bf16" else 4
        gate, vectors = case["gates"] * D * size, 4 * D * sum({"": 0, "rms": 1, "layer": 2}[case[k]] for k in ("post", "pre"))
        nbytes = 2 * M * D * (size + stream) + gate + vectors          # read h, x, gate; write x', y
        if case["train"]:
            nbytes += 2 * M * D * (size + stream) + gate + vectors     # read the gradients of x', y; write those of h, x and the rest
        return {"bytes": nbytes, "flops": (40.0 if case["train"] else 12.0) * M * D}
    n = sum(math.prod(shape) for shape in _gradient_shapes(case))
    return {"bytes": n * size + (4 * n if case["clip"] else 0), "flops": (3.0 if case["clip"] else 2.0) * n}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_layer(case, s):
    rows = []
    w = s["w"].double().t().contiguous()
    for at in range(0, case["rows"], 16384):
        part = slice(at, at + 16384)
        if case["op"] == "layer":
            x = s["x"][part].double()
            top = x.abs().amax(dim=1, keepdim=True)
            a, scale = torch.round(x * 127.0 / torch.clamp(top, min=1e-300)), top / 127.0
        else:
            a, scale = s["a"][part].double(), s["a_scale"][part].double()[:, None]
        v = torch.mm(a, w) * (scale * s["w_scale"].double()[None, :])
        if s["bias"] is not None:
            v += s["bias"].double()
        if s["residual"] is not None:
            v += s["residual"][part].double()
        rows.append(v * torch.sigmoid(v) if case["act"] else v)
    return torch.cat(rows)


def _exact_norm(v, kind, weight, bias):
    """(the norm, its unscaled form, 1 / its deviation) in 64 bits"""
    centred = v - v.sum(dim=1, keepdim=True) / v.shape[1] if kind == "layer" else v
    inverse = (centred.pow(2).sum(dim=1, keepdim=True) / v.shape[1] + EPS).pow(-0.5)
    unit = centred * inverse
    return unit * weight.double() + (0.0 if bias is None else bias.double()), unit, inverse


def _exact_norm_backward(grad, kind, weight, unit, inverse):
    """gradients of (input, weight, bias) by the formula d v = (g - [mean g] - unit * mean(g * unit)) / deviation, g = grad * weight"""
    g = grad * weight.double()
    d = g - unit * (g * unit).mean(dim=1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(dim=1, keepdim=True)
    return d * inverse, (grad * unit).sum(dim=0), grad.sum(dim=0)


def _exact_residual_norm(case, s):
    M, G, scale = case["rows"], case["gates"], case["residual_scale"]
    h, x = s["h"].detach().double(), s["x"].detach().double()
    row_gate = torch.arange(M, device="cuda") // (M // G)
    gate = s["gate"].detach().double()
    u = h
    if case["post"]:
        u, post_unit, post_inverse = _exact_norm(h, case["post"], s["post_weight"].detach(), None if s["post_bias"] is None else s["post_bias"].detach())
    new = scale * x + gate[row_gate] * u
    y, unit, inverse = _exact_norm(new, case["pre"], s["pre_weight"].detach(), None if s["pre_bias"] is None else s["pre_bias"].detach())
    if not case["train"]:
        return {"x": new, "y": y}
    d, d_pre_weight, d_pre_bias = _exact_norm_backward(s["grad_y"].double(), case["pre"], s["pre_weight"].detach(), unit, inverse)
    d += s["grad_x"].double()
    grads = {"x": scale * d, "gate": (d * u).view(G, M // G, -1).sum(dim=1), "pre_weight": d_pre_weight, "pre_bias": d_pre_bias}
    grads["h"] = d * gate[row_gate]
    if case["post"]:
        grads["h"], grads["post_weight"], grads["post_bias"] = _exact_norm_backward(grads["h"], case["post"], s["post_weight"].detach(), post_unit, post_inverse)
    return {"x": new, "y": y, "grads": {k: grads[k] for k in s["leaves"]}}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("product", "layer"):
        return _exact_layer(case, s)
    if case["op"] == "norm":
        return _exact_residual_norm(case, s)
    total = sum(float((g.double() ** 2).sum()) for g in s["grads"])
    norm = torch.tensor(math.sqrt(total), dtype=torch.float64)
    if not case["clip"]:
        return norm
    factor = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    return {"norm": norm, "clipped": torch.cat([g.double().reshape(-1) * factor for g in s["grads"]])}
