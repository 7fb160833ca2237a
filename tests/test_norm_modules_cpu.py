"""Which path the model's LayerNorm takes, decided without a GPU (the kernels' calls are replaced)."""
import pytest
import torch

from dcnv4_b200 import flash_intern_image as fii
from dcnv4_b200 import ops


@pytest.mark.parametrize("weight,bias,x", [(w, b, x) for w in (False, True) for b in (False, True) for x in (False, True)])
def test_the_inference_kernel_runs_only_where_nothing_learns(weight, bias, x, monkeypatch):
    """It records no graph, so a bias that learns beside a frozen weight has to keep it away."""
    ln = fii.LayerNorm(8)
    ln.weight.requires_grad_(weight)
    ln.bias.requires_grad_(bias)
    taken = []
    monkeypatch.setattr(ops, "layer_norm_supported", lambda *a: True)
    monkeypatch.setattr(ops, "layer_norm_forward", lambda t, *a: taken.append(1) or t.detach())
    y = ln(torch.randn(2, 8, requires_grad=x))
    learns = weight or bias or x
    assert bool(taken) == (not learns) and y.requires_grad == learns
    with torch.no_grad():
        ln(torch.randn(2, 8))
    assert taken


@pytest.mark.parametrize("learns", ["none", "x", "weight", "bias", "residual", "norm weight", "norm bias"])
def test_the_fused_linear_runs_only_where_nothing_learns(learns, monkeypatch):
    """Its bias, the residual it adds and the LayerNorm in its epilogue count as much as its weight."""
    F = torch.nn.functional
    lin, norm = torch.nn.Linear(8, 8).requires_grad_(False), torch.nn.LayerNorm(8).requires_grad_(False)
    x, residual = torch.randn(4, 8), torch.randn(4, 8)
    leaf = {"none": None, "x": x, "weight": lin.weight, "bias": lin.bias, "residual": residual, "norm weight": norm.weight,
            "norm bias": norm.bias}[learns]
    if leaf is not None:
        leaf.requires_grad_(True)

    def plain(t, w, b, r=None, act="none"):
        return (F.linear(t, w, b) + r).detach()

    monkeypatch.setattr(ops, "linear_supported", lambda *a: True)
    monkeypatch.setattr(ops, "_norm_fusable", lambda *a: True)
    monkeypatch.setattr(ops, "LN_FUSION_MIN_ROWS_PER_SM", 0)
    monkeypatch.setattr(ops, "_sm_count", lambda d: 1)
    monkeypatch.setattr(ops, "linear_forward", plain)
    monkeypatch.setattr(ops, "linear_layer_norm_forward",
                        lambda t, w, b, r, nw, nb, eps: (plain(t, w, b, r), F.layer_norm(plain(t, w, b, r), (8,), nw, nb, eps).detach()))
    y, z = ops.linear_module_forward(x, lin, residual, norm=norm)
    assert z.requires_grad == (leaf is not None)
    assert y.requires_grad == (leaf is not None and not learns.startswith("norm"))
    if leaf is not None:
        z.square().sum().backward()
        assert leaf.grad is not None


# ---- what stands beside the norms --------------------------------------------------------------------------

class Halve(torch.nn.Module):
    def forward(self, x):
        return 0.5 * x


class LoudDropPath(fii.DropPath):
    def forward(self, x):
        return 3.0 * x


class ShiftedNorm(fii.LayerNorm):
    def forward(self, x):
        return super().forward(x) + 1.0


def _patched():
    m = torch.nn.Identity()
    m.forward = lambda x: 2.0 * x
    return m


def _hooked():
    m = torch.nn.Identity()
    m.register_forward_hook(lambda mod, args, out: 4.0 * out)
    return m


@pytest.fixture
def kernels(monkeypatch):
    """The library's functions, replaced by their formulas: records which were taken, with the plain results."""
    taken = []
    F = torch.nn.functional

    def post(x, res, w, b, eps, gamma=None, s=None):
        taken.append("post")
        z = F.layer_norm(x, (x.shape[-1],), w, b, eps) * (1.0 if gamma is None else gamma)
        return res + (z if s is None else z * s.view(-1, *[1] * (x.dim() - 1)))

    def pre(x, res, w, b, eps, s=None):
        taken.append("pre")
        h = res + (x if s is None else x * s.view(-1, *[1] * (x.dim() - 1)))
        return h, F.layer_norm(h, (x.shape[-1],), w, b, eps)

    monkeypatch.setattr(fii.LayerNorm, "train_out_dtype", lambda self, x: x.dtype)
    monkeypatch.setattr(fii.LayerNorm, "forward_act", lambda self, x, activation="none": None)
    monkeypatch.setattr(fii.LayerNormResidualFunction, "apply", post)
    monkeypatch.setattr(fii.AddLayerNormFunction, "apply", pre)
    return taken


@pytest.mark.parametrize("make,fused", [(torch.nn.Identity, True), (lambda: fii.DropPath(0.0), True), (lambda: fii.DropPath(0.5), True),
                                        (Halve, False), (lambda: torch.nn.Dropout(0.5), False), (lambda: LoudDropPath(0.5), False),
                                        (_patched, False), (_hooked, False)],
                         ids=["identity", "drop path 0", "drop path", "another module", "dropout", "subclass", "own forward", "hook"])
def test_what_replaces_the_drop_path_is_called(make, fused, kernels):
    norm = fii.build_norm_layer(8, "LN")
    x, res = torch.randn(4, 3, 8), torch.randn(4, 3, 8)
    for run, which in ((lambda d: fii._post_norm(norm, x, res, None, d), "post"), (lambda d: fii._pre_norm(norm, x, res, d), "pre")):
        kernels.clear()
        torch.manual_seed(3)
        got = run(make())
        assert (which in kernels) == fused
        torch.manual_seed(3)
        drop = make()
        want = res + drop(norm(x)) if which == "post" else (lambda h: (h, norm(h)))(res + drop(x))
        torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)


def test_norms_that_compute_something_else_are_called(kernels):
    x, res = torch.randn(4, 8), torch.randn(4, 8)
    for norm in (ShiftedNorm(8), torch.nn.Sequential(ShiftedNorm(8))):
        torch.testing.assert_close(fii._post_norm(norm, x, res, None, torch.nn.Identity()), res + norm(x))
        torch.testing.assert_close(fii._pre_norm(norm, x, res, torch.nn.Identity()), (res + x, norm(res + x)))
    assert not kernels


@pytest.mark.parametrize("register", ["register_module_forward_hook", "register_module_forward_pre_hook",
                                      "register_module_full_backward_hook"])
def test_hooks_of_all_modules_see_the_calls(register, kernels):
    from torch.nn.modules import module as nn_module
    norm = fii.build_norm_layer(8, "LN")
    x, res = torch.randn(4, 8, requires_grad=True), torch.randn(4, 8)
    handle = getattr(nn_module, register)(lambda *a: None)
    try:
        fii._post_norm(norm, x, res, None, torch.nn.Identity())
        fii._pre_norm(norm, x, res, torch.nn.Identity())
        assert not kernels
    finally:
        handle.remove()
    fii._post_norm(norm, x, res, None, torch.nn.Identity())
    assert kernels == ["post"]


def test_the_stem_calls_hooked_and_replaced_modules(monkeypatch):
    """Its norm and activation run as one kernel only where both are what the stem was built with."""
    taken = []
    monkeypatch.setattr(fii.LayerNorm, "forward_act", lambda self, x, activation="none":
                        taken.append(activation) or torch.nn.functional.gelu(self._stock(x)) if activation == "gelu" else None)
    monkeypatch.setattr(fii.LayerNorm, "_stock", torch.nn.LayerNorm.forward, raising=False)
    x = torch.randn(1, 3, 16, 16)

    class OtherGELU(torch.nn.GELU):
        def forward(self, t):
            return torch.zeros_like(t)

    for change in ("none", "norm hook", "layer hook", "act hook", "act class", "norm class"):
        torch.manual_seed(0)
        stem = fii.StemLayer(3, 16, "GELU", "LN")
        seen = []
        if change == "norm hook":
            stem.norm1.register_forward_hook(lambda *a: seen.append(1))
        elif change == "layer hook":
            stem.norm1[1].register_forward_pre_hook(lambda *a: seen.append(1))
        elif change == "act hook":
            stem.act.register_forward_hook(lambda *a: seen.append(1))
        elif change == "act class":
            stem.act = OtherGELU()
        elif change == "norm class":
            stem.norm1[1] = ShiftedNorm(8)
        taken.clear()
        out = stem(x)
        assert bool(taken) == (change == "none"), change
        assert bool(seen) == change.endswith("hook"), change
        if change == "act class":
            torch.testing.assert_close(out, stem.norm2(stem.conv2(torch.zeros(1, 8, 8, 8))).contiguous())


# ---- tensors and modes that only the stock operations support ------------------------------------------------

def test_fake_tensors_train_through_the_stock_operation():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True):
        ln = fii.LayerNorm(8, device="cuda")
        x = torch.empty(4, 8, device="cuda", requires_grad=True)
        y = ln(x)
        assert y.shape == (4, 8) and "LayerNorm" in y.grad_fn.name()
        h, z = fii._pre_norm(ln, x, x, torch.nn.Identity())
        assert z.shape == h.shape == (4, 8)
        assert fii._post_norm(ln, x, x, None, torch.nn.Identity()).shape == (4, 8)


def test_kernels_decline_what_they_cannot_see_through():
    from torch.utils._python_dispatch import TorchDispatchMode
    from dcnv4_b200.functions.layer_norm_func import kernels_apply

    class Tagged(torch.Tensor):
        pass

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x = torch.zeros(2, 8)
    assert kernels_apply(x, None, torch.nn.Parameter(x))
    assert not kernels_apply(x, x.as_subclass(Tagged))
    with Watch():
        assert not kernels_apply(x)
    seen = []
    torch.func.vmap(lambda t: seen.append(kernels_apply(t)) or t)(x)
    torch.jit.trace(lambda t: seen.append(kernels_apply(t)) or t, (x,), check_trace=False)
    assert not any(seen) and len(seen) >= 2
    assert kernels_apply(x)
