"""The training-step operators as a model uses them: FlashInternImage with the library's norms against the stock
modules, the Muon optimiser against its formulas in 64 bits, and a few steps of both together."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tiny(**kw):
    from dcnv4_b200 import flash_intern_image as fii
    torch.manual_seed(0)
    cfg = dict(channels=32, depths=(1, 2, 2, 1), groups=(2, 4, 8, 16), num_classes=10, offset_scale=1.0)
    cfg.update(kw)
    return fii.FlashInternImage(**cfg).to(DEV).train()


CONFIGS = {
    "pre-norm": dict(drop_path_rate=0.0),
    "pre-norm, stochastic depth": dict(drop_path_rate=0.5),
    "pre-norm, layer scale": dict(drop_path_rate=0.3, layer_scale=0.5),
    "post-norm": dict(drop_path_rate=0.0, post_norm=True),
    "post-norm, layer scale, stochastic depth": dict(drop_path_rate=0.5, post_norm=True, layer_scale=0.5),
    "checkpointed": dict(drop_path_rate=0.3, post_norm=True, layer_scale=0.5, with_cp=True),
}


def step(model, x, labels, library, autocast=None):
    from dcnv4_b200.flash_intern_image import LayerNorm
    LayerNorm.use_library_kernel = library
    try:
        torch.manual_seed(7)                       # the stochastic-depth masks
        with torch.autocast("cuda", dtype=autocast or torch.bfloat16, enabled=autocast is not None):
            loss = torch.nn.functional.cross_entropy(model(x).float(), labels)
        model.zero_grad(set_to_none=True)
        loss.backward()
        return loss.detach(), {k: p.grad for k, p in model.named_parameters()}
    finally:
        LayerNorm.use_library_kernel = True


@pytest.mark.parametrize("name", list(CONFIGS))
def test_model_gradients_equal_the_stock_modules(name, monkeypatch):
    """Same masks, same loss, same gradients: library norms and stock norms in fp32.  The two differ by fp32 roundings,
    which the layers amplify: 1e-3 of a gradient's norm is 2^14 roundings."""
    from dcnv4_b200 import ops
    model = tiny(**CONFIGS[name])
    x = torch.randn(4, 3, 64, 96, device=DEV)
    labels = torch.randint(0, 10, (4,), device=DEV)
    calls = []
    for fn in ("layer_norm_backward", "layer_norm_residual_backward", "add_layer_norm_backward"):
        inner = getattr(ops, fn)
        monkeypatch.setattr(ops, fn, lambda *a, _f=fn, _i=inner, **k: (calls.append(_f), _i(*a, **k))[1])
    tf32 = torch.backends.cudnn.allow_tf32
    torch.backends.cudnn.allow_tf32 = False
    try:
        loss, got = step(model, x, labels, True)
        used = set(calls)
        n = len(calls)
        want_loss, want = step(model, x, labels, False)
        assert len(calls) == n                     # the stock run took none of them
    finally:
        torch.backends.cudnn.allow_tf32 = tf32
    assert "layer_norm_backward" in used
    assert ("layer_norm_residual_backward" in used) == ("post" in name or name == "checkpointed")
    assert ("add_layer_norm_backward" in used) == name.startswith("pre-norm, ")
    torch.testing.assert_close(loss, want_loss, rtol=1e-4, atol=1e-5)
    for k in want:
        assert (got[k] is None) == (want[k] is None), k
        if want[k] is not None:
            assert got[k].dtype == want[k].dtype
            assert (got[k] - want[k]).norm() <= 1e-3 * want[k].norm() + 1e-6, k


@pytest.mark.parametrize("name", ["pre-norm, stochastic depth", "post-norm, layer scale, stochastic depth"])
def test_model_trains_under_autocast_and_in_bf16(name):
    x = torch.randn(4, 3, 64, 96, device=DEV)
    labels = torch.randint(0, 10, (4,), device=DEV)
    model = tiny(**CONFIGS[name])
    loss, got = step(model, x, labels, True, torch.bfloat16)
    want_loss, want = step(model, x, labels, False, torch.bfloat16)
    # both runs round every product to bf16: 2^-8 a rounding, some dozens of them between a weight and the loss
    assert abs(float(loss - want_loss)) < 64 * 2.0 ** -8
    for k in want:
        assert torch.isfinite(got[k]).all() and got[k].dtype == torch.float32, k
    half = copy.deepcopy(model).bfloat16()
    loss, got = step(half, x.bfloat16(), labels, True)
    assert torch.isfinite(loss) and all(torch.isfinite(g).all() for g in got.values())


def test_norms_keep_what_the_stock_module_does():
    """Second derivatives, torch.func transforms, forward-mode AD, hooks and mixed types behave as with nn.LayerNorm."""
    from dcnv4_b200.flash_intern_image import LayerNorm, _pre_norm
    ln = LayerNorm(24, eps=1e-6).to(DEV)
    ref = torch.nn.LayerNorm(24, eps=1e-6).to(DEV)
    x = torch.randn(5, 24, device=DEV, requires_grad=True)
    outs = []
    for m in (ln, ref):
        (g,) = torch.autograd.grad((m(x) ** 3).sum(), x, create_graph=True)
        outs.append(torch.autograd.grad((g ** 2).sum(), x)[0])
    torch.testing.assert_close(outs[0], outs[1], rtol=1e-3, atol=1e-3)
    f = torch.func.grad(lambda t: (ln(t) ** 2).sum())
    torch.testing.assert_close(f(x.detach()), torch.func.grad(lambda t: (ref(t) ** 2).sum())(x.detach()), rtol=1e-4, atol=1e-4)
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        y = ln(fwad.make_dual(x.detach(), torch.ones_like(x)))
        assert fwad.unpack_dual(y).tangent is not None
    seen = []
    handle = ln.register_forward_hook(lambda *a: seen.append(1))
    _pre_norm(ln, x, x, torch.nn.Identity())
    handle.remove()
    assert seen
    with pytest.raises(RuntimeError):
        ln(x.half())
    t = x.detach().t().contiguous().t().requires_grad_(True)      # not contiguous
    ln(t).sum().backward()
    assert t.grad.shape == t.shape


# ------------------------------------------------------------------------------------------- Muon

def ns64(x, steps=5):
    a, b, c = 3.4445, -4.7750, 2.0315
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        A = x @ x.T
        x = a * x + (b * A + c * A @ A) @ x
    return x.T if tall else x


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", ["match_rms_adamw", "original"])
def test_muon_follows_its_formulas(nesterov, adjust):
    """Three steps over shapes that form stacks of one and of several, a convolution among them.  The update is good to
    4.8e-3 of its norm (see the orthogonalisation's own test); a step adds it scaled by lr, the buffers stay fp32."""
    from dcnv4_b200 import Muon
    g = torch.Generator(device=DEV).manual_seed(0)
    shapes = [(48, 64), (48, 64), (64, 48), (48, 64), (40, 24, 3, 3)]
    params = [torch.nn.Parameter(torch.randn(s, device=DEV, generator=g)) for s in shapes]
    params[4].data = params[4].data.contiguous(memory_format=torch.channels_last)
    lr, wd, mu = 0.02, 0.1, 0.9
    opt = Muon(params, lr=lr, weight_decay=wd, momentum=mu, nesterov=nesterov, adjust_lr=adjust)
    want = [p.detach().double().clone() for p in params]
    bufs = [torch.zeros_like(w) for w in want]
    slack = [0.0] * len(params)
    for _ in range(3):
        for i, p in enumerate(params):
            p.grad = torch.randn(shapes[i], device=DEV, generator=g)
            bufs[i] = mu * bufs[i] + (1 - mu) * p.grad.double()
            u = mu * bufs[i] + (1 - mu) * p.grad.double() if nesterov else bufs[i]
            rows, cols = shapes[i][0], math.prod(shapes[i][1:])
            o = ns64(u.reshape(rows, cols)).view(shapes[i])
            s = 0.2 * math.sqrt(max(rows, cols)) if adjust == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))
            want[i] = (1 - lr * wd) * want[i] - lr * s * o
            slack[i] += lr * s * 4.8e-3 * float(o.norm())
        opt.step()
    for p, w, b, sl in zip(params, want, bufs, slack):
        assert float((p.detach().double() - w).norm()) <= sl + 8 * 2.0 ** -24 * float(w.norm())
        torch.testing.assert_close(opt.state[p]["momentum_buffer"].double(), b, rtol=1e-5, atol=1e-6)


def test_muon_state_dict_and_refusals():
    from dcnv4_b200 import Muon
    from dcnv4_b200.muon import split_parameters
    w = torch.nn.Parameter(torch.randn(16, 24, device=DEV))
    opt = Muon([w], lr=0.01)
    w.grad = torch.randn_like(w)
    opt.step()
    other = Muon([torch.nn.Parameter(w.detach().clone())], lr=0.5)
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["lr"] == 0.01
    torch.testing.assert_close(next(iter(other.state.values()))["momentum_buffer"], opt.state[w]["momentum_buffer"])
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(ns_steps=0), dict(adjust_lr="none")):
        with pytest.raises(ValueError):
            Muon([w], **bad)
    with pytest.raises(ValueError, match="vectors"):
        Muon([torch.nn.Parameter(torch.zeros(4, device=DEV))])
    model = tiny()
    matrices, others = split_parameters(model)
    assert all(p.dim() >= 2 for p in matrices)
    assert len(matrices) + len(others) == len(list(model.parameters()))
    assert any(p is model.head.weight for p in others)


def test_a_training_step_with_all_of_them():
    """Norms forward and backward, stochastic depth, layer scale and the Muon step, as a trainer runs them."""
    from dcnv4_b200 import Muon
    from dcnv4_b200.muon import split_parameters
    model = tiny(drop_path_rate=0.3, post_norm=True, layer_scale=0.1)
    matrices, others = split_parameters(model)
    opts = [Muon(matrices, lr=1e-3), torch.optim.AdamW(others, lr=1e-3)]
    x = torch.randn(4, 3, 64, 64, device=DEV)
    labels = torch.randint(0, 10, (4,), device=DEV)
    before = [p.detach().clone() for p in model.parameters()]
    for _ in range(3):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = torch.nn.functional.cross_entropy(model(x).float(), labels)
        for o in opts:
            o.zero_grad(set_to_none=True)
        loss.backward()
        for o in opts:
            o.step()
    assert torch.isfinite(loss)
    for (name, p), b in zip(model.named_parameters(), before):
        assert torch.isfinite(p).all(), name
        assert not torch.equal(p, b), name
