"""LayerNorm training passes (plain, post-norm tail, pre-norm seam) against 64-bit formulas.

Tolerances.  Sums run in fp32: a lane adds at most 48 elements before at most 9 levels of reduction, so a row sum is off
by at most 64 * 2^-24 of the sum of magnitudes.  The mean's error shifts every element, so the normalised value is off by
64 * 2^-24 * (1 + max|x| rstd) (kappa below), and what is linear in it by that times its factor.  A column sum adds at
most rows / 148 + 96 terms in sequence.  The final rounding adds half a step of the storage type, and a stored `h` another
half step of the value that the backward pass normalises.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]
IDS = ["f32", "f16", "bf16", "f16-f32", "bf16-f32"]
EPS = 1e-6
U = 2.0 ** -24
SHAPES = [(1, 1), (3, 2), (5, 7), (1, 8), (49, 64), (130, 80), (33, 161), (64, 160), (9, 640), (1000, 32), (6, 1003),
          (7, 1280), (2, 4096), (5, 8192), (4, 8191)]


def half_step(t):
    return torch.finfo(t).eps / 2 if t != F32 else 0.0


def make(rows, C, tx, ty, tw, seed=0, samples=1, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 1000 * rows + C)

    def randn(*s):
        return torch.randn(*s, device=DEV, generator=g)

    def place(t):
        if not offset:
            return t
        flat = torch.empty(t.numel() + offset, dtype=t.dtype, device=DEV)
        out = flat[offset:].view(t.shape)
        return out.copy_(t)

    d = {"x": place((randn(rows, C) * 1.5 + 0.7).to(tx)), "res": place(randn(rows, C).to(ty)),
         "w": place((1 + 0.3 * randn(C)).to(tw)), "b": place((0.3 * randn(C)).to(tw)),
         "gamma": place((0.5 * randn(C)).to(tw)), "gy": place(randn(rows, C).to(ty)), "gh": place(randn(rows, C).to(ty))}
    d["s"] = None
    if samples > 1:
        keep = torch.rand(samples, device=DEV, generator=g) < 0.7
        keep[0], keep[-1] = False, True          # always one dropped and one kept sample
        d["s"] = keep.float() / 0.7
    return d


def ref(mode, d, act="none", s=True):
    """64-bit forward values and gradients, and the magnitudes the tolerances need."""
    x, res, w, b, gamma, gy, gh = (d[k].double() for k in ("x", "res", "w", "b", "gamma", "gy", "gh"))
    rows, C = x.shape
    f = d["s"].double().repeat_interleave(rows // d["s"].numel())[:, None] if s and d["s"] is not None else 1.0
    v = res + f * x if mode == "pre" else x
    mean = v.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + EPS)
    xh = (v - mean) * rstd
    z = xh * w + b
    g, we = gy, w
    o = {}
    if mode == "post":
        o["y"] = res + f * gamma * z
        g, we = f * gy, w * gamma
    elif act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        o["y"] = z * cdf
        g = gy * (cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
    else:
        o["y"] = z
    gw = g * we
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    A, B = (g * xh).sum(0), g.sum(0)
    absA, absB = (g * xh).abs().sum(0), g.abs().sum(0)
    if mode == "post":
        o |= {"gx": dx, "gw": gamma * A, "gb": gamma * B, "gs": w * A + b * B}
    elif mode == "pre":
        o |= {"h": v, "gr": dx + gh, "gx": f * (dx + gh), "gw": A, "gb": B}
    else:
        o |= {"gx": dx, "gw": A, "gb": B}
    kappa = 1 + v.abs().amax(1, keepdim=True) * rstd
    xm = 1 + xh.abs().amax(1, keepdim=True)
    o["_xh_err"] = 64 * U * kappa * xm
    o["_dx_err"] = 64 * U * kappa * rstd * xm ** 2 * (gw.abs().amax(1, keepdim=True) if C else 0) * 4
    n = rows / 148 + 96
    o["_A_err"] = n * U * absA + (64 * U * kappa * xm * g.abs()).sum(0)
    o["_B_err"] = n * U * absB
    o["_rstd"], o["_xm"], o["_gwmax"], o["_g"], o["_v"] = rstd, xm, gw.abs().amax(1, keepdim=True), g, v
    o["_f"] = f
    return o


def within(got, want, err, what):
    diff = (got.double() - want).abs()
    bad = ~(diff <= err)
    assert not bool(bad.any()), f"{what}: off by {diff[bad].max().item():.3g} (allowed {torch.as_tensor(err, device=diff.device).expand_as(diff)[bad].min().item():.3g}) at {int(bad.sum())} places"


def rounded(want, err, t):
    """Allowed distance once `want` (itself off by `err`) is rounded to t: half a step, at least the subnormals'."""
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 if t != F32 else 0.0
    return err + half_step(t) * (want.abs() + err) + tiny


def check_params(o, got, d, mode, rows):
    tw = d["w"].dtype
    w, b, gamma = d["w"].double(), d["b"].double(), d["gamma"].double()
    if mode == "post":
        errs = {"gw": gamma.abs() * o["_A_err"], "gb": gamma.abs() * o["_B_err"],
                "gs": w.abs() * o["_A_err"] + b.abs() * o["_B_err"]}
    else:
        errs = {"gw": o["_A_err"], "gb": o["_B_err"]}
    for k, e in errs.items():
        assert got[k].dtype == tw and got[k].shape == w.shape
        within(got[k], o[k], rounded(o[k], e + 4 * U * o[k].abs(), tw), k)


def run_plain(d, act="none"):
    from dcnv4_b200 import ops
    y, m, r = ops.layer_norm_train_forward(d["x"], d["w"], d["b"], EPS, act, d["gy"].dtype)
    gx, gw, gb = ops.layer_norm_backward(d["gy"], d["x"], m, r, d["w"], d["b"], act)
    return {"y": y, "gx": gx, "gw": gw, "gb": gb}


def run_post(d, scale=True):
    from dcnv4_b200 import ops
    gamma = d["gamma"] if scale else None
    y, m, r = ops.layer_norm_residual_forward(d["x"], d["res"], d["w"], d["b"], EPS, gamma, d["s"])
    gx, gw, gb, gs = ops.layer_norm_residual_backward(d["gy"], d["x"], m, r, d["w"], d["b"], gamma, d["s"])
    return {"y": y, "gx": gx, "gw": gw, "gb": gb, "gs": gs}


def run_pre(d, gh=True):
    from dcnv4_b200 import ops
    h, y, m, r = ops.add_layer_norm_forward(d["x"], d["res"], d["w"], d["b"], EPS, d["s"])
    gr, gx, gw, gb = ops.add_layer_norm_backward(d["gy"], d["gh"] if gh else None, h, m, r, d["w"], d["s"], d["x"].dtype)
    return {"h": h, "y": y, "gr": gr, "gx": gx, "gw": gw, "gb": gb}


def check_plain(d, act="none"):
    tx, ty = d["x"].dtype, d["gy"].dtype
    got, o = run_plain(d, act), ref("plain", d, act)
    wmax = d["w"].double().abs()
    ye = o["_xh_err"] * wmax + 4 * U * (o["y"].abs() + d["b"].double().abs())
    de = o["_dx_err"]
    if act == "gelu":
        # |d gelu / dz| <= 1.13 and |d gelu' / dz| <= 0.8; erff and expf are good to a few steps of values <= 1
        ye = 1.2 * ye + 8 * U * (1 + o["y"].abs())
        zerr = (o["_xh_err"] * wmax + 4 * U * (1 + d["b"].double().abs()) + 16 * U) * d["gy"].double().abs() * wmax
        de = de + 3 * o["_rstd"] * o["_xm"] ** 2 * zerr.amax(1, keepdim=True)
        ge = 0.8 * (o["_xh_err"] * wmax + 4 * U * (1 + d["b"].double().abs())) * d["gy"].double().abs() + 16 * U * d["gy"].double().abs()
        o["_A_err"] = o["_A_err"] + (ge * o["_xm"]).sum(0)
        o["_B_err"] = o["_B_err"] + ge.sum(0)
    assert got["y"].dtype == ty and got["gx"].dtype == tx
    within(got["y"], o["y"], rounded(o["y"], ye, ty), "y")
    within(got["gx"], o["gx"], rounded(o["gx"], de, tx), "gx")
    check_params(o, got, d, "plain", d["x"].shape[0])


def check_post(d, scale=True):
    tx, ty = d["x"].dtype, d["gy"].dtype
    e = dict(d) if scale else dict(d, gamma=torch.ones_like(d["gamma"]))
    got, o = run_post(d, scale), ref("post", e)
    we = (d["w"].double() * e["gamma"].double()).abs() + (d["b"].double() * e["gamma"].double()).abs()
    f = o["_f"]
    ye = (f * o["_xh_err"] if torch.is_tensor(f) else o["_xh_err"]) * we + 6 * U * (o["y"].abs() + 2 * we * o["_xm"] + d["res"].double().abs())
    within(got["y"], o["y"], rounded(o["y"], ye, ty), "out")
    within(got["gx"], o["gx"], rounded(o["gx"], o["_dx_err"], tx), "gx")
    if not scale:
        assert got["gs"] is None
        o["_A_err"], o["_B_err"] = o["_A_err"], o["_B_err"]
        for k in ("gw", "gb"):
            err = o["_A_err"] if k == "gw" else o["_B_err"]
            within(got[k], o[k], rounded(o[k], err + 4 * U * o[k].abs(), d["w"].dtype), k)
    else:
        check_params(o, got, d, "post", d["x"].shape[0])


def check_pre(d, gh=True):
    tx, ty = d["x"].dtype, d["gy"].dtype
    e = dict(d) if gh else dict(d, gh=torch.zeros_like(d["gh"]))
    got, o = run_pre(d, gh), ref("pre", e)
    within(got["h"], o["h"], rounded(o["h"], 2 * U * (o["h"].abs() + 3 * d["x"].double().abs()), ty), "h")
    ye = (o["_xh_err"]) * d["w"].double().abs() + 4 * U * (o["y"].abs() + d["b"].double().abs())
    within(got["y"], o["y"], rounded(o["y"], ye, ty), "y")
    # the backward pass normalises the stored h, half a step of which moves xh by hd
    hd = half_step(ty) * o["_v"].abs().amax(1, keepdim=True) * o["_rstd"]
    de = o["_dx_err"] + 4 * o["_rstd"] * o["_gwmax"] * hd * (o["_xm"] + hd)
    de = de + 4 * U * e["gh"].double().abs()
    within(got["gr"], o["gr"], rounded(o["gr"], de, ty), "gr")
    f = o["_f"]
    fe = f * de if torch.is_tensor(f) else de
    within(got["gx"], o["gx"], rounded(o["gx"], fe + 2 * U * o["gx"].abs(), tx), "gx")
    assert got["gx"].dtype == tx and got["gr"].dtype == ty and got["h"].dtype == ty
    o["_A_err"] = o["_A_err"] + (hd * d["gy"].double().abs()).sum(0)
    check_params(o, got, d, "pre", d["x"].shape[0])


@pytest.mark.parametrize("tx,ty", PAIRS, ids=IDS)
@pytest.mark.parametrize("rows,C", SHAPES)
def test_plain(rows, C, tx, ty):
    for tw in {F32, tx}:
        check_plain(make(rows, C, tx, ty, tw))


@pytest.mark.parametrize("tx,ty", PAIRS, ids=IDS)
@pytest.mark.parametrize("rows,C", [(49, 32), (130, 80), (5, 7), (6, 1003), (3, 2048)])
def test_plain_with_gelu(rows, C, tx, ty):
    check_plain(make(rows, C, tx, ty, F32), "gelu")


@pytest.mark.parametrize("tx,ty", PAIRS, ids=IDS)
@pytest.mark.parametrize("rows,C,samples", [(1, 8, 1), (48, 64, 3), (130, 80, 2), (6, 1003, 3), (64, 160, 64), (4, 8192, 2),
                                            (9, 1, 3), (300, 640, 4)])
def test_post(rows, C, samples, tx, ty):
    d = make(rows, C, tx, ty, F32 if rows % 4 else tx, samples=samples)
    check_post(d)
    check_post(d, scale=False)


@pytest.mark.parametrize("tx,ty", PAIRS, ids=IDS)
@pytest.mark.parametrize("rows,C,samples", [(1, 8, 1), (48, 64, 3), (130, 80, 2), (6, 1003, 3), (64, 160, 64), (4, 8192, 2),
                                            (9, 1, 3), (300, 640, 4)])
def test_pre(rows, C, samples, tx, ty):
    d = make(rows, C, tx, ty, F32 if rows % 4 else tx, samples=samples)
    check_pre(d)
    check_pre(d, gh=False)


@pytest.mark.parametrize("tx,ty", PAIRS, ids=IDS)
def test_many_rows(tx, ty):
    """Enough rows for every CTA to walk several, in teams of a few lanes, a warp and a CTA."""
    for rows, C in ((40001, 24), (20011, 256), (3001, 1536)):
        d = make(rows, C, tx, ty, F32)
        check_plain(d)
        check_pre(d)
        check_post(d)


@pytest.mark.parametrize("tx,ty", PAIRS, ids=IDS)
def test_unaligned_tensors(tx, ty):
    """Views one element into their storage: no row starts on a vector boundary."""
    for C in (64, 72, 1024):
        d = make(12, C, tx, ty, F32, samples=3, offset=1)
        check_plain(d)
        check_post(d)
        check_pre(d)


@pytest.mark.parametrize("C", [8192, 8191])
def test_offsets_beyond_32_bits(C):
    """More than 2^32 elements: the last rows against the same rows on their own."""
    from dcnv4_b200 import ops
    rows, tail = 2 ** 32 // C + 1500, 700
    if torch.cuda.mem_get_info()[0] < 50 << 30:
        pytest.skip("needs 50 GB")
    g = torch.Generator(device=DEV).manual_seed(11)
    x = torch.zeros(rows, C, device=DEV, dtype=BF16)
    x[-tail:] = torch.randn(tail, C, device=DEV, generator=g)
    w, b = (torch.randn(C, device=DEV, generator=g) for _ in range(2))
    y, mean, rstd = ops.layer_norm_train_forward(x, w, b, EPS)
    gx, gw, gb = ops.layer_norm_backward(x, x, mean, rstd, w, b)
    own = x[-tail:].clone()
    want, m, r = ops.layer_norm_train_forward(own, w, b, EPS)
    assert torch.equal(y[-tail:], want) and torch.equal(mean[-tail:], m) and torch.equal(rstd[-tail:], r)
    wx, ww, wb = ops.layer_norm_backward(own, own, m, r, w, b)
    assert torch.equal(gx[-tail:], wx)
    assert torch.equal(y[0], b.to(BF16)) and not gx[:1000].any()
    # parameter gradients: other rows are zero, so both are sums of the same values in other orders
    scale = own.double().abs().sum(0)
    order = 2 * tail * 2.0 ** -24                        # each of two orders of `tail` fp32 additions
    assert bool(((gb - wb).double().abs() <= order * scale).all())
    xh = (own.double() - m[:, None]) * r[:, None]
    assert bool(((gw - ww).double().abs() <= 1.01 * order * (xh * own.double()).abs().sum(0)).all())


def test_degenerate_rows():
    """Constant rows have no spread: xh is 0 and rstd 1/sqrt(eps); the gradient follows the formula."""
    d = make(6, 40, F32, F32, F32)
    d["x"][2] = 3.25
    d["x"][4] = 0.0
    got = run_plain(d)
    torch.testing.assert_close(got["y"][2], d["b"])
    torch.testing.assert_close(got["y"][4], d["b"])
    o = ref("plain", d)
    torch.testing.assert_close(got["gx"].double(), o["gx"], rtol=1e-4, atol=1e-3 / math.sqrt(EPS) * 1e-3)


def test_no_rows():
    from dcnv4_b200 import ops
    for tw in (F32, BF16):
        x = torch.empty(0, 48, device=DEV, dtype=BF16)
        w = torch.ones(48, device=DEV, dtype=tw)
        y, m, r = ops.layer_norm_train_forward(x, w, w, EPS)
        assert y.shape == (0, 48) and m.shape == (0,)
        gx, gw, gb = ops.layer_norm_backward(y, x, m, r, w, w)
        assert gx.shape == (0, 48) and not gw.any() and not gb.any() and gw.dtype == tw
        gs = ops.layer_norm_residual_backward(y, x, m, r, w, w, w, torch.empty(0, device=DEV))[3]
        assert not gs.any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_row_stays_in_its_row(bad):
    """NaN or infinity in one row of x reaches that row's outputs and the parameter gradients, no other row."""
    for C in (24, 160, 1003, 4096):
        d = make(9, C, F32, F32, F32)
        good = run_pre(d)
        d["x"][4, C // 2] = bad
        got = run_pre(d)
        rows = [r for r in range(9) if r != 4]
        for k in ("h", "y", "gr", "gx"):
            assert torch.equal(got[k][rows], good[k][rows])
        assert not torch.isfinite(got["y"][4]).any() and got["gw"].isnan().any()


def test_repeats_bit_for_bit():
    for C in (80, 161, 2048):
        d = make(4099, C, BF16, F32, F32)
        for fn in (run_plain, run_post, run_pre):
            a, b = fn(d), fn(d)
            assert all(torch.equal(a[k], b[k]) for k in a)


def test_rows_behind_the_last_are_left_alone():
    """Outputs are written for the given rows only: guard rows around the storage keep their values."""
    from dcnv4_b200 import _lib
    L = _lib.lib()
    rows, C = 13, 72
    d = make(rows, C, F16, F32, F32)

    def guarded(shape, dtype):
        n = math.prod(shape)
        full = torch.full((n + 64,), 7.0, dtype=dtype, device=DEV)
        return full, full[32:32 + n].view(shape)

    fy, y = guarded((rows, C), F32)
    fm, m = guarded((rows,), F32)
    fr, r = guarded((rows,), F32)
    stream = torch.cuda.current_stream().cuda_stream
    assert L.dcnv4b200_layernorm_train_fwd(d["x"].data_ptr(), None, d["w"].data_ptr(), d["b"].data_ptr(), None, None,
                                           y.data_ptr(), None, m.data_ptr(), r.data_ptr(), 0, _lib.F16, _lib.F32,
                                           _lib.F32, rows, C, rows, EPS, 0, stream) == 0
    fx, gx = guarded((rows, C), F16)
    fw, gw = guarded((C,), F32)
    fb, gb = guarded((C,), F32)
    need = L.dcnv4b200_layernorm_train_bwd_workspace_bytes(_lib.F16, rows, C)
    fs, ws = guarded((need // 4,), F32)
    assert L.dcnv4b200_layernorm_train_bwd(d["gy"].data_ptr(), None, d["x"].data_ptr(), m.data_ptr(), r.data_ptr(),
                                           d["w"].data_ptr(), d["b"].data_ptr(), None, None, gx.data_ptr(), None,
                                           gw.data_ptr(), gb.data_ptr(), None, ws.data_ptr(), need, 0, _lib.F16,
                                           _lib.F32, _lib.F32, rows, C, rows, 0, stream) == 0
    want = run_plain(d)
    for full, view, key in ((fy, y, "y"), (fx, gx, "gx"), (fw, gw, "gw"), (fb, gb, "gb"), (fm, m, None), (fr, r, None),
                            (fs, ws, None)):
        assert (full[:32] == 7).all() and (full[32 + view.numel():] == 7).all()
        if key:
            assert torch.equal(view, want[key])


def test_another_stream_and_a_captured_graph():
    d = make(513, 96, BF16, F32, F32, samples=3)
    want = run_post(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_post(d)
    side.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)
    graphs = []
    for _ in range(2):                                  # two graphs of the same calls, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            static = run_post(d)
        graphs.append((graph, static))
    d["x"].mul_(1.25)
    want = run_post(d)
    for graph, static in graphs * 2:
        graph.replay()
        assert all(torch.equal(static[k], want[k]) for k in want)


def test_captured_backward_pass():
    """Forward and backward of the three functions as one captured graph, replayed after its inputs changed."""
    from dcnv4_b200 import AddLayerNormFunction, LayerNormFunction, LayerNormResidualFunction
    g = torch.Generator(device=DEV).manual_seed(3)
    leaves = [torch.randn(shape, device=DEV, generator=g, requires_grad=True)
              for shape in ((4, 50, 192), (4, 50, 192), (192,), (192,))]

    def grads():
        x, r, w, b = leaves
        h, y = AddLayerNormFunction.apply(x, r, w, b, 1e-6)
        z = LayerNormFunction.apply(y, w, b, 1e-6, "gelu")
        loss = LayerNormResidualFunction.apply(z, h, w, b, 1e-6, w).square().mean()
        return torch.autograd.grad(loss, leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = grads()
    with torch.no_grad():
        for t in leaves:
            t.mul_(1.5)
    graph.replay()
    for a, b in zip(static, grads()):
        assert torch.equal(a, b)


def test_directional_differences():
    """The gradients against central differences of the kernel's own forward pass, in fp32.  Allowed: the forward's
    rounding over the step, and the truncation that the 64-bit formula shows for the same step."""
    from dcnv4_b200 import ops
    for mode in ("plain", "gelu", "post", "pre"):
        d = make(6, 24, F32, F32, F32, samples=3)
        step = 2.0 ** -6
        for name in ("x", "w", "b") + (("gamma",) if mode == "post" else ()) + (("res",) if mode in ("post", "pre") else ()):
            v = torch.randn_like(d[name])
            v /= v.norm()

            def loss(sign, exact):
                e = dict(d)
                e[name] = d[name] + sign * step * v if not exact else d[name].double() + sign * step * v.double()
                if exact:
                    o = ref("plain" if mode == "gelu" else mode, e, "gelu" if mode == "gelu" else "none")
                    return (o["y"] * d["gy"].double()).sum() + ((o["h"] * d["gh"].double()).sum() if mode == "pre" else 0)
                if mode == "pre":
                    h, y, _, _ = ops.add_layer_norm_forward(e["x"], e["res"], e["w"], e["b"], EPS, e["s"])
                    return (y.double() * d["gy"].double()).sum() + (h.double() * d["gh"].double()).sum()
                if mode == "post":
                    y = ops.layer_norm_residual_forward(e["x"], e["res"], e["w"], e["b"], EPS, e["gamma"], e["s"])[0]
                else:
                    y = ops.layer_norm_train_forward(e["x"], e["w"], e["b"], EPS, "gelu" if mode == "gelu" else "none")[0]
                return (y.double() * d["gy"].double()).sum()

            got = run_pre(d) if mode == "pre" else run_post(d) if mode == "post" else run_plain(d, "gelu" if mode == "gelu" else "none")
            grad = {"x": got["gx"], "w": got["gw"], "b": got["gb"], "gamma": got.get("gs"),
                    "res": got.get("gr", d["gy"])}[name]
            o = ref("plain" if mode == "gelu" else mode, d, "gelu" if mode == "gelu" else "none")
            exact = {"x": o["gx"], "w": o["gw"], "b": o["gb"], "gamma": o.get("gs"), "res": o.get("gr", d["gy"].double())}[name]
            slope = (loss(1, False) - loss(-1, False)).item() / (2 * step)
            truth = (loss(1, True) - loss(-1, True)).item() / (2 * step)
            along = (grad.double() * v.double()).sum().item()
            truncation = abs(truth - (exact * v.double()).sum().item())
            # every output is good to 64 (1 + kappa) steps; the perturbed input itself rounds once
            rounding = 256 * U * 8 * float(d["gy"].abs().sum() + d["gh"].abs().sum()) / step
            assert abs(slope - along) <= truncation + rounding, (mode, name, slope, along, truncation, rounding)


def test_autograd_functions_match_the_stock_modules():
    """The three functions inside autograd, with broadcast and non-contiguous gradients, against stock PyTorch in fp32."""
    from dcnv4_b200.functions import AddLayerNormFunction, LayerNormFunction, LayerNormResidualFunction
    F = torch.nn.functional
    N, L, C = 3, 20, 64
    d = make(N * L, C, F32, F32, F32, samples=N)

    def leaves():
        return [d[k].clone().requires_grad_(True) for k in ("x", "res", "w", "b", "gamma")]

    s = d["s"].view(N, 1, 1)
    for which in ("plain", "post", "pre"):
        grads = []
        for lib in (True, False):
            x, res, w, b, gamma = leaves()
            x3, r3 = x.view(N, L, C), res.view(N, L, C)
            if which == "plain":
                y = LayerNormFunction.apply(x3, w, b, EPS) if lib else F.layer_norm(x3, (C,), w, b, EPS)
                out = y.transpose(1, 2)[:, ::2].sum(1)                # a strided, broadcast gradient
            elif which == "post":
                out = (LayerNormResidualFunction.apply(x3, r3, w, b, EPS, gamma, d["s"]) if lib
                       else r3 + s * gamma * F.layer_norm(x3, (C,), w, b, EPS))
            else:
                h, y = AddLayerNormFunction.apply(x3, r3, w, b, EPS, d["s"]) if lib else (None, None)
                if not lib:
                    h = r3 + s * x3
                    y = F.layer_norm(h, (C,), w, b, EPS)
                out = torch.cat([h * 0.5, y], -1)
            (out * out).sum().backward()
            grads.append([t.grad for t in (x, res, w, b, gamma)])
        for a, b_ in zip(*grads):
            assert (a is None) == (b_ is None)
            if a is not None:
                torch.testing.assert_close(a, b_, rtol=1e-4, atol=1e-4)


def test_only_one_output_of_the_seam_is_used():
    from dcnv4_b200.functions import AddLayerNormFunction
    d = make(10, 32, F32, F32, F32)
    for pick in (0, 1):
        x, res = d["x"].clone().requires_grad_(True), d["res"].clone().requires_grad_(True)
        w = d["w"].clone().requires_grad_(True)
        out = AddLayerNormFunction.apply(x, res, w, d["b"], EPS)
        out[pick].backward(d["gy"])
        x2, r2, w2 = (t.detach().clone().requires_grad_(True) for t in (x, res, w))
        h = r2 + x2
        (h if pick == 0 else torch.nn.functional.layer_norm(h, (32,), w2, d["b"], EPS)).backward(d["gy"])
        torch.testing.assert_close(x.grad, x2.grad, rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(res.grad, r2.grad, rtol=1e-5, atol=1e-5)
        if pick:
            torch.testing.assert_close(w.grad, w2.grad, rtol=1e-5, atol=1e-5)


def test_refusals():
    from dcnv4_b200 import ops
    x = torch.randn(4, 16, device=DEV)
    w = torch.ones(16, device=DEV)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.layer_norm_train_forward(x.t(), w[:4], w[:4], EPS)
    with pytest.raises(RuntimeError, match="size of the last"):
        ops.layer_norm_train_forward(x, w[:8], w[:8], EPS)
    with pytest.raises(RuntimeError, match="dtype"):
        ops.layer_norm_train_forward(x, w.half(), w.half(), EPS)
    with pytest.raises(RuntimeError, match="dtype"):
        ops.layer_norm_train_forward(x, w, w, EPS, "none", torch.float16)
    with pytest.raises(ValueError):
        ops.layer_norm_train_forward(x, w, w, EPS, "relu")
    with pytest.raises(ValueError):
        big = torch.zeros(1, 8193, device=DEV)
        ops.layer_norm_train_forward(big, big[0], big[0], EPS)
    with pytest.raises(RuntimeError, match="shape"):
        ops.layer_norm_residual_forward(x, x[:2], w, w, EPS)
    with pytest.raises(RuntimeError, match="sample_scale"):
        ops.layer_norm_residual_forward(x, x, w, w, EPS, None, torch.ones(3, device=DEV))
    with pytest.raises(RuntimeError, match="sample_scale"):
        ops.add_layer_norm_forward(x, x, w, w, EPS, torch.ones(4, device=DEV).half())
    y, m, r = ops.layer_norm_train_forward(x, w, w, EPS)
    with pytest.raises(RuntimeError, match="statistics"):
        ops.layer_norm_backward(y, x, m[:2].contiguous(), r, w, w)
    with pytest.raises(RuntimeError, match="float64|supports"):
        ops.layer_norm_train_forward(x.double(), w.double(), w.double(), EPS)


@pytest.mark.parametrize("tx,ty", PAIRS, ids=IDS)
@pytest.mark.parametrize("C", [3, 9, 12, 20, 33, 62, 100, 129, 250, 515, 1001, 1004, 1010, 1011, 1018, 2042, 2044, 4094])
def test_widths_no_vector_divides(C, tx, ty):
    """Every distance of a row's start from a vector boundary, a last tile that ends inside one, one sample per few rows."""
    for rows, samples in ((8, 2), (333, 3), (1500 if C < 600 else 40, 4)):
        d = make(rows, C, tx, ty, F32 if rows % 2 else tx, samples=samples)
        check_plain(d)
        check_post(d)
        check_pre(d)
    check_plain(make(37, C, tx, ty, F32), "gelu")
