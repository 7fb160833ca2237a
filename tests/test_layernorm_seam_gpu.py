"""The pre-norm seam in 16 bits: its backward pass belongs to its forward.

Statistics and y are those of the fp32 sum, and so are the gradients: nothing here grants the rounding of the stored h.
Tolerances are those of `test_layernorm_train_gpu` without that term: fp32 sums, and half a step where a result is
stored in 16 bits.  A row's kappa = 1 + max|h| / sigma is large where its spread is small, and the bound with it.
"""
import pytest
import torch

from tests.test_layernorm_train_gpu import (BF16, DEV, EPS, F16, F32, U, check_params, half_step, make, ref, rounded, within)

pytestmark = pytest.mark.gpu
HALVES = pytest.mark.parametrize("t", [F16, BF16], ids=["f16", "bf16"])


def run(d, gh=True):
    from dcnv4_b200 import ops
    h, y, m, r = ops.add_layer_norm_forward(d["x"], d["res"], d["w"], d["b"], EPS, d["s"])
    gr, gx, gw, gb = ops.add_layer_norm_backward(d["gy"], d["gh"] if gh else None, h, m, r, d["w"], d["s"], None, d["x"],
                                                 d["res"])
    return {"h": h, "y": y, "gr": gr, "gx": gx, "gw": gw, "gb": gb}


def check(d, gh=True, got=None):
    t = d["x"].dtype
    got = run(d, gh) if got is None else got
    o = ref("pre", d if gh else dict(d, gh=torch.zeros_like(d["gh"])))
    if "y" in got:
        ye = o["_xh_err"] * d["w"].double().abs() + 4 * U * (o["y"].abs() + d["b"].double().abs())
        within(got["y"], o["y"], rounded(o["y"], ye, t), "y")
        within(got["h"], o["h"], rounded(o["h"], 2 * U * (o["h"].abs() + 3 * d["x"].double().abs()), t), "h")
    de = o["_dx_err"] + 4 * U * (d["gh"].double().abs() if gh else 0.0)
    within(got["gr"], o["gr"], rounded(o["gr"], de, t), "gr")
    f = o["_f"]
    fe = f * de if torch.is_tensor(f) else de
    within(got["gx"], o["gx"], rounded(o["gx"], fe + 2 * U * o["gx"].abs(), t), "gx")
    check_params(o, got, d, "pre", d["x"].shape[0])


@HALVES
@pytest.mark.parametrize("rows,C,samples", [(1, 1, 1), (1, 8, 1), (48, 64, 3), (130, 80, 2), (6, 1003, 3), (64, 160, 64), (4, 8192, 2),
                                            (9, 1, 3), (300, 640, 4), (333, 33, 3), (40, 2042, 4), (40001, 24, 1), (20011, 256, 1)])
def test_gradients_are_those_at_the_sum(rows, C, samples, t):
    for tw in (F32, t):
        d = make(rows, C, t, t, tw, samples=samples)
        check(d)
        check(d, gh=False)
    if rows < 1000:                      # no row on a vector boundary: the element-wise kernels
        check(make(rows, C, t, t, F32, samples=samples, offset=1))


def flat_rows(C, t, offset=0):
    """Rows whose spread is nothing, or small beside a rounding step of the stored sum, and ordinary ones between them."""
    d = make(12, C, t, t, F32, samples=3, offset=offset)
    d["s"] = torch.tensor([1.0, 0.5, 2.0], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(C)
    for row, spread in ((0, 0.0), (3, 0.0), (5, 1e-4), (10, 1e-3), (11, 0.0)):
        d["res"][row] = 1.0 if row != 11 else 100.0
        d["x"][row] = (0.003 + spread * torch.randn(C, device=DEV, generator=g)).to(t)
    return d


@HALVES
@pytest.mark.parametrize("C", [8, 40, 128, 1003, 4096])
def test_rows_with_little_spread(C, t):
    for offset in (0, 1):
        check(flat_rows(C, t, offset))


@HALVES
@pytest.mark.parametrize("C", [8, 40, 128, 1003, 4096])
def test_from_the_stored_sum_alone(C, t):
    """Without x and residual: h as stored, its own mean, and the smaller of the given 1/sigma and its own."""
    from dcnv4_b200 import ops
    for offset in (0, 1):
        d = flat_rows(C, t, offset)
        h, y, m, r = ops.add_layer_norm_forward(d["x"], d["res"], d["w"], d["b"], EPS, d["s"])
        if offset:
            h = make(12, C, t, t, F32, offset=1)["x"].copy_(h)
        gr, gx, gw, gb = ops.add_layer_norm_backward(d["gy"], d["gh"], h, m, r, d["w"], d["s"])
        v, gy, w = h.double(), d["gy"].double(), d["w"].double()
        own = v.var(1, unbiased=False, keepdim=True)
        rstd = torch.minimum(r.double()[:, None], torch.where(own > 0, own, 0.0).rsqrt())
        xh = (v - v.mean(1, keepdim=True)) * rstd
        xm = 1 + xh.abs().amax(1, keepdim=True)
        kappa = 1 + v.abs().amax(1, keepdim=True) * rstd
        gv = gy * w
        dx = rstd * (gv - gv.mean(1, keepdim=True) - xh * (gv * xh).mean(1, keepdim=True)) + d["gh"].double()
        err = 4 * 64 * U * kappa * rstd * xm ** 2 * gv.abs().amax(1, keepdim=True) + 4 * U * d["gh"].double().abs()
        within(gr, dx, rounded(dx, err, t), "gr")
        f = d["s"].double().repeat_interleave(4)[:, None]
        within(gx, f * dx, rounded(f * dx, f * err + 2 * U * (f * dx).abs(), t), "gx")
        A, B = (gy * xh).sum(0), gy.sum(0)
        within(gw, A, 108 * U * (gy * xh).abs().sum(0) + (64 * U * kappa * xm * gy.abs()).sum(0) + 4 * U * A.abs(), "gw")
        within(gb, B, 112 * U * gy.abs().sum(0), "gb")
        # constant rows: nothing reaches the weight's gradient (a 64-bit mean of C equal values up to 100 is off by at
        # most C * 2^-53 * 100 <= 4.6e-11, times 1/sigma <= 1000)
        assert xh[[0, 11]].abs().max() <= 4.6e-8


@HALVES
def test_the_two_routes_into_the_library_agree(t, monkeypatch):
    """The C binding and the Python route behind it."""
    from dcnv4_b200 import ops

    class Declines:
        ln_forward = ln_backward = staticmethod(lambda *a: None)

    d = make(130, 72, t, t, F32, samples=2)
    want = run(d)
    monkeypatch.setattr(ops, "_binding", Declines)
    got = run(d)
    assert all(torch.equal(got[k], want[k]) for k in want)


@HALVES
def test_autograd_function_and_its_second_derivative(t):
    """The function's gradients, the same gradients under create_graph, and the gradient of one of them."""
    from dcnv4_b200.functions import AddLayerNormFunction
    d = flat_rows(48, t)
    names = ("x", "res", "w", "b")

    def leaves():
        return [d[k].clone().requires_grad_(True) for k in names]

    for create in (False, True):
        x, res, w, b = leaves()
        out = AddLayerNormFunction.apply(x, res, w, b, EPS, d["s"])
        gx, gr, gw, gb = torch.autograd.grad(out, (x, res, w, b), (d["gh"], d["gy"]), create_graph=create)
        check(d, got={"gx": gx.detach(), "gr": gr.detach(), "gw": gw.detach(), "gb": gb.detach()})
    # along v, differentiated again; ordinary rows, where kappa is a few
    d = make(12, 48, t, t, F32, samples=3)
    v = torch.randn(12, 48, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(t)
    x, res, w, b = leaves()
    out = AddLayerNormFunction.apply(x, res, w, b, EPS, d["s"])
    (gr,) = torch.autograd.grad(out, res, (d["gh"], d["gy"]), create_graph=True)
    got = torch.autograd.grad(gr, (x, res, w), v)
    x, res, w, b = (d[k].double().requires_grad_(True) for k in names)
    h = res + d["s"].double().repeat_interleave(4)[:, None] * x
    y = torch.nn.functional.layer_norm(h, (48,), w, b, EPS)
    (gr,) = torch.autograd.grad((h, y), res, (d["gh"].double(), d["gy"].double()), create_graph=True)
    want = torch.autograd.grad(gr, (x, res, w), v.double())
    for a, e in zip(got, want):
        # some ten row sums in fp32 over values up to the largest, then one rounding
        within(a, e, rounded(e, 10 * 64 * 8 * U * e.abs().max(), a.dtype), "second derivative")


def test_streams_graphs_and_repetition():
    d = make(513, 96, BF16, BF16, F32, samples=3)
    want = run(d)
    assert all(torch.equal(a, b) for a, b in zip(run(d).values(), want.values()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = run(d)
    d["x"].mul_(1.25)
    graph.replay()
    want = run(d)
    assert all(torch.equal(static[k], want[k]) for k in want)


def test_refusals():
    from dcnv4_b200 import ops
    d = make(6, 16, BF16, BF16, F32)
    h, y, m, r = ops.add_layer_norm_forward(d["x"], d["res"], d["w"], d["b"], EPS)
    args = (d["gy"], None, None, m, r, d["w"], None)
    for kw in (dict(), dict(x=d["x"]), dict(residual=d["res"]), dict(x=d["x"], residual=d["res"][:3]),
               dict(x=d["x"], residual=d["res"].half()), dict(x=d["x"].half(), residual=d["res"]),
               dict(x=d["x"], residual=d["res"].t().contiguous().t()), dict(x=d["x"], residual=d["res"], x_dtype=F32)):
        with pytest.raises(RuntimeError):
            ops.add_layer_norm_backward(*args, **kw)
    f = make(6, 16, BF16, F32, F32)                       # fp32 h: x and residual are not needed, and do not replace it
    h, y, m, r = ops.add_layer_norm_forward(f["x"], f["res"], f["w"], f["b"], EPS)
    with pytest.raises(RuntimeError):
        ops.add_layer_norm_backward(f["gy"], None, None, m, r, f["w"], None, BF16, f["x"], f["res"])
    a = ops.add_layer_norm_backward(f["gy"], None, h, m, r, f["w"], None, BF16, f["x"], f["res"])
    b = ops.add_layer_norm_backward(f["gy"], None, h, m, r, f["w"], None, BF16)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    e = make(6, 16, BF16, BF16, F32)
    empty = torch.empty(0, 16, device=DEV, dtype=BF16)
    none = torch.empty(0, device=DEV)
    gr, gx, gw, gb = ops.add_layer_norm_backward(empty, None, None, none, none, e["w"], None, None, empty, empty)
    assert gr.shape == (0, 16) and not gw.any() and not gb.any()
