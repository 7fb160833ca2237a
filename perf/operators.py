"""Workloads of the training-step operators: LayerNorm with its gradient, in the three places a FlashInternImage
layer has it, and the Newton-Schulz orthogonalisation of a weight matrix' update.

    layer_norm           y = act(LN(x)); act is nothing or the exact GELU; x may be narrower than y (autocast)
    layer_norm_residual  out = residual + s * gamma * LN(x): the tail of a post-norm block, with the layer scale
                         gamma (C) and the stochastic-depth factor s (one number per sample)
    add_layer_norm       h = residual + s * x, y = LN(h): the seam between two pre-norm branches
    newton_schulz        X0 = G / (|G|_F + eps), then five times X <- a X + (b A + c A A) X with A = X X^T; bf16 out

The first three are a forward and a backward pass each; `own` selects the library's calls or the plain formulas.
"""
import math

import torch

own = False

EPS = 1e-6
NS = (3.4445, -4.7750, 2.0315)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the last stage of FlashInternImage-T (224 x 224) for one image: 7 x 7 tokens, the call's latency
        {"name": "ln one image f32", "op": "layer_norm", "rows": 49, "C": 512, "x": "f32", "y": "f32", "w": "f32",
         "act": "none", "samples": 1},
        # the stem's first norm with its GELU, 64 images of 112 x 112 in fp16
        {"name": "ln stem gelu f16", "op": "layer_norm", "rows": 64 * 112 * 112, "C": 32, "x": "f16", "y": "f16",
         "w": "f16", "act": "gelu", "samples": 64},
        # stage 1 of FlashInternImage-L at 1024 x 1024, two images under bf16 autocast: bf16 in, fp32 out
        {"name": "ln stage1 autocast", "op": "layer_norm", "rows": 2 * 256 * 256, "C": 160, "x": "bf16", "y": "f32",
         "w": "f32", "act": "none", "samples": 2},
        # a width that no vector divides, in bf16
        {"name": "ln odd width bf16", "op": "layer_norm", "rows": 9973, "C": 1003, "x": "bf16", "y": "bf16",
         "w": "bf16", "act": "none", "samples": 1},
        # the post-norm block of FlashInternImage-L's long third stage, two images under autocast
        {"name": "post stage3 autocast", "op": "layer_norm_residual", "rows": 2 * 64 * 64, "C": 640, "x": "bf16",
         "y": "f32", "w": "f32", "act": "none", "samples": 2},
        # stage 1 of FlashInternImage-S (224 x 224) in pure bf16, 64 images
        {"name": "post stage1 bf16", "op": "layer_norm_residual", "rows": 64 * 56 * 56, "C": 80, "x": "bf16",
         "y": "bf16", "w": "bf16", "act": "none", "samples": 64},
        # the seam of a pre-norm FlashInternImage-T block, second stage, 64 images in fp16
        {"name": "pre stage2 f16", "op": "add_layer_norm", "rows": 64 * 28 * 28, "C": 128, "x": "f16", "y": "f16",
         "w": "f16", "act": "none", "samples": 64},
        # wide fp32 rows (a head-sized width), few of them
        {"name": "pre wide f32", "op": "add_layer_norm", "rows": 2048, "C": 4096, "x": "f32", "y": "f32", "w": "f32",
         "act": "none", "samples": 8},
        # the value projection of FlashInternImage-T's first stage, alone: the call's latency
        {"name": "ns 64x64", "op": "newton_schulz", "batch": 1, "m": 64, "n": 64, "x": "f32", "y": "bf16"},
        # the classifier of FlashInternImage-T, taller than wide, rows that no tile divides
        {"name": "ns head 1000x768", "op": "newton_schulz", "batch": 1, "m": 1000, "n": 768, "x": "f32", "y": "bf16"},
        # fc2 of all layers of FlashInternImage-L's third stage, stacked
        {"name": "ns stage3 fc2", "op": "newton_schulz", "batch": 22, "m": 640, "n": 2560, "x": "f32", "y": "bf16"},
        # fc1 of all layers of its last stage, stacked and tall, momentum kept in bf16
        {"name": "ns stage4 fc1", "op": "newton_schulz", "batch": 5, "m": 5120, "n": 1280, "x": "bf16", "y": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "layer_norm_residual", "add_layer_norm", "newton_schulz",
                     "newton_schulz"])
    if op == "newton_schulz":
        while True:
            p, q = sorted((_log(rng, 16, 1280), _log(rng, 16, 5120)))
            batch = _log(rng, 1, 24)
            if p > 1280 or batch * p * q > 16 * 2 ** 20:
                continue
            m, n = (p, q) if rng.random() < 0.5 else (q, p)
            return {"op": op, "batch": batch, "m": m, "n": n, "x": rng.choice(["f32", "f32", "bf16", "f16"]),
                    "y": "bf16"}
    C = _log(rng, 8, 4096)
    if rng.random() < 0.7:
        C = max(8, C // 8 * 8)
    samples = rng.choice([1, 2, 8, 64])
    most = {"layer_norm": 15, "layer_norm_residual": 12, "add_layer_norm": 8}[op] * 2 ** 20
    rows = samples * _log(rng, 1, max(1, most // (C * samples)))
    x, y = rng.choice([("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
    w = y if rng.random() < 0.5 else "f32"
    if w != "f32" and w != x:
        w = "f32"
    act = "gelu" if op == "layer_norm" and rng.random() < 0.25 else "none"
    return {"op": op, "rows": rows, "C": C, "x": x, "y": y, "w": w, "act": act, "samples": samples}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "newton_schulz":
        # a momentum buffer: a few strong directions over the gradient's noise, at a gradient's scale
        B, m, n = case["batch"], case["m"], case["n"]
        r = max(1, min(m, n) // 16)
        G = randn(B, m, r) @ randn(B, r, n) / math.sqrt(r) + 0.1 * randn(B, m, n)
        return {"case": case, "x": (G * 1e-3).to(TYPES[case["x"]])}
    rows, C, S = case["rows"], case["C"], case["samples"]
    tx, ty, tw = TYPES[case["x"]], TYPES[case["y"]], TYPES[case["w"]]

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    # activations: every channel with a mean and a spread of its own
    s = {"case": case,
         "x": (randn(rows, C) * (0.5 + rand(C)) + 0.5 * randn(C)).to(tx),
         "weight": (0.5 + rand(C)).to(tw), "bias": (0.3 * randn(C)).to(tw),
         "grad": (0.1 * randn(rows, C)).to(ty)}
    if case["op"] != "layer_norm":
        s["residual"] = (randn(rows, C) + 0.2 * randn(C)).to(ty)
        # stochastic depth: a sample's branch is dropped with probability 0.1, else scaled up
        s["sample_scale"] = ((rand(S) >= 0.1).float() / 0.9) if S > 1 else None
    if case["op"] == "layer_norm_residual":
        s["layer_scale"] = (0.05 + 0.45 * rand(C)).to(tw)
    if case["op"] == "add_layer_norm":
        s["grad_h"] = (0.1 * randn(rows, C)).to(ty)
    return s


def _per_row(sample_scale, rows):
    return sample_scale.repeat_interleave(rows // sample_scale.numel())[:, None] if sample_scale is not None else 1.0


def _normalised(x):
    """The normalised rows and 1 / sigma, in 32 bits."""
    d = x - x.mean(1, keepdim=True)
    rstd = ((d * d).mean(1, keepdim=True) + EPS).rsqrt()
    return d * rstd, rstd


def _grad_rows(gw, xhat, rstd):
    return rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))


def _plain(s):
    case = s["case"]
    ty = TYPES[case["y"]]
    if case["op"] == "newton_schulz":
        a, b, c = NS
        x = s["x"].float()
        tall = case["m"] > case["n"]
        x = x.transpose(1, 2) if tall else x
        x = x / (x.double().square().sum((1, 2), keepdim=True).sqrt().float() + 1e-7)
        for _ in range(5):
            A = x @ x.transpose(1, 2)
            x = a * x + (b * A + c * (A @ A)) @ x
        return {"out": (x.transpose(1, 2) if tall else x).to(ty)}
    x, w, b, gy = s["x"].float(), s["weight"].float(), s["bias"].float(), s["grad"].float()
    tx, tw = s["x"].dtype, s["weight"].dtype
    if case["op"] == "layer_norm":
        xhat, rstd = _normalised(x)
        z = xhat * w + b
        y = z
        if case["act"] == "gelu":
            cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
            y = z * cdf
            gy = gy * (cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
        return {"y": y.to(ty), "grad_x": _grad_rows(gy * w, xhat, rstd).to(tx),
                "grad_weight": (gy * xhat).sum(0).to(tw), "grad_bias": gy.sum(0).to(tw)}
    f = _per_row(s["sample_scale"], case["rows"])
    if case["op"] == "layer_norm_residual":
        gamma = s["layer_scale"].float()
        xhat, rstd = _normalised(x)
        z = xhat * w + b
        gz = f * gy
        return {"out": (s["residual"].float() + f * gamma * z).to(ty),
                "grad_x": _grad_rows(gz * gamma * w, xhat, rstd).to(tx),
                "grad_weight": (gz * gamma * xhat).sum(0).to(tw), "grad_bias": (gz * gamma).sum(0).to(tw),
                "grad_layer_scale": (gz * z).sum(0).to(tw)}
    h = s["residual"].float() + f * x
    hhat, rstd = _normalised(h)
    gh = _grad_rows(gy * w, hhat, rstd) + s["grad_h"].float()
    return {"h": h.to(ty), "y": (hhat * w + b).to(ty), "grad_residual": gh.to(ty), "grad_x": (f * gh).to(tx),
            "grad_weight": (gy * hhat).sum(0).to(tw), "grad_bias": gy.sum(0).to(tw)}


def _own(s):
    from dcnv4_b200 import ops
    case = s["case"]
    if case["op"] == "newton_schulz":
        return {"out": ops.newton_schulz(s["x"], steps=5, coefficients=NS, eps=1e-7)}
    if case["op"] == "layer_norm":
        y, mean, rstd = ops.layer_norm_train_forward(s["x"], s["weight"], s["bias"], EPS, case["act"],
                                                     out_dtype=TYPES[case["y"]])
        gx, gw, gb = ops.layer_norm_backward(s["grad"], s["x"], mean, rstd, s["weight"], s["bias"], case["act"])
        return {"y": y, "grad_x": gx, "grad_weight": gw, "grad_bias": gb}
    if case["op"] == "layer_norm_residual":
        out, mean, rstd = ops.layer_norm_residual_forward(s["x"], s["residual"], s["weight"], s["bias"], EPS,
                                                          s["layer_scale"], s["sample_scale"])
        gx, gw, gb, gs = ops.layer_norm_residual_backward(s["grad"], s["x"], mean, rstd, s["weight"], s["bias"],
                                                          s["layer_scale"], s["sample_scale"])
        return {"out": out, "grad_x": gx, "grad_weight": gw, "grad_bias": gb, "grad_layer_scale": gs}
    h, y, mean, rstd = ops.add_layer_norm_forward(s["x"], s["residual"], s["weight"], s["bias"], EPS,
                                                  s["sample_scale"])
    # a 16-bit h has lost bits of the sum that was normalised: the pass forms it again from branch and residual
    gr, gx, gw, gb = ops.add_layer_norm_backward(s["grad"], s["grad_h"], h, mean, rstd, s["weight"],
                                                 s["sample_scale"], s["x"].dtype, s["x"], s["residual"])
    return {"h": h, "y": y, "grad_residual": gr, "grad_x": gx, "grad_weight": gw, "grad_bias": gb}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    sx, sy = size[case["x"]], size[case["y"]]
    if case["op"] == "newton_schulz":
        p, q = sorted((case["m"], case["n"]))
        # A and A A are symmetric: half of their products suffice
        return {"bytes": case["batch"] * p * q * (sx + sy), "flops": 5 * case["batch"] * (3 * p * p * q + p ** 3)}
    sw = size[case["w"]]
    e, C = case["rows"] * case["C"], case["C"]
    if case["op"] == "layer_norm":        # x, grad in; y, grad_x out
        return {"bytes": e * (2 * sx + 2 * sy) + 4 * C * sw, "flops": 20 * e}
    if case["op"] == "layer_norm_residual":  # x, residual, grad in; out, grad_x out
        return {"bytes": e * (2 * sx + 3 * sy) + 6 * C * sw, "flops": 24 * e}
    # x, residual, grad, grad_h in; h, y, grad_residual, grad_x out
    return {"bytes": e * (2 * sx + 6 * sy) + 4 * C * sw, "flops": 24 * e}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "newton_schulz":
        # the iteration on the Gram matrix alone: with M = a I + G (b I + c G), P <- M P and G <- M G M, the
        # result is P X0 (all of these are polynomials in X0 X0^T and commute)
        a, b, c = NS
        x = s["x"].double()
        tall = case["m"] > case["n"]
        if tall:
            x = x.mT.contiguous()
        x = x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)
        G = torch.bmm(x, x.mT)
        eye = torch.eye(G.shape[1], dtype=torch.float64, device=x.device).expand_as(G)
        P = eye
        for _ in range(5):
            M = a * eye + torch.bmm(G, b * eye + c * G)
            P = torch.bmm(M, P)
            G = torch.bmm(torch.bmm(M, G), M)
        y = torch.bmm(P, x)
        return {"out": y.mT if tall else y}
    F = torch.nn.functional
    leaf = {k: v.double().requires_grad_(True) for k, v in s.items()
            if isinstance(v, torch.Tensor) and not k.startswith("grad") and k != "sample_scale"}
    gy = s["grad"].double()
    C = case["C"]
    if case["op"] == "layer_norm":
        y = F.layer_norm(leaf["x"], (C,), leaf["weight"], leaf["bias"], EPS)
        y = F.gelu(y) if case["act"] == "gelu" else y
        gx, gw, gb = torch.autograd.grad(y, (leaf["x"], leaf["weight"], leaf["bias"]), gy)
        return {"y": y, "grad_x": gx, "grad_weight": gw, "grad_bias": gb}
    branch = leaf["x"]
    if case["op"] == "layer_norm_residual":
        branch = F.layer_norm(branch, (C,), leaf["weight"], leaf["bias"], EPS) * leaf["layer_scale"]
    if s["sample_scale"] is not None:
        per = s["sample_scale"].double()
        branch = (branch.view(per.numel(), -1, C) * per.view(-1, 1, 1)).view(-1, C)
    h = leaf["residual"] + branch
    if case["op"] == "layer_norm_residual":
        gx, gw, gb, gs = torch.autograd.grad(h, (leaf["x"], leaf["weight"], leaf["bias"], leaf["layer_scale"]), gy)
        return {"out": h, "grad_x": gx, "grad_weight": gw, "grad_bias": gb, "grad_layer_scale": gs}
    y = F.layer_norm(h, (C,), leaf["weight"], leaf["bias"], EPS)
    gr, gx, gw, gb = torch.autograd.grad((h, y), (leaf["residual"], leaf["x"], leaf["weight"], leaf["bias"]),
                                         (s["grad_h"].double(), gy))
    return {"h": h, "y": y, "grad_residual": gr, "grad_x": gx, "grad_weight": gw, "grad_bias": gb}
