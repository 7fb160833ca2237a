"""The model's LayerNorm as a module on the GPU: which inputs train, what stands around it, how they lie in memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pair(C, **trained):
    """The library's module and the stock one with the same parameters; `trained` says which of them learn."""
    from dcnv4_b200.flash_intern_image import LayerNorm
    torch.manual_seed(C)
    mods = [LayerNorm(C, eps=1e-6).to(DEV), torch.nn.LayerNorm(C, eps=1e-6).to(DEV)]
    with torch.no_grad():
        mods[0].weight.uniform_(0.5, 1.5)
        mods[0].bias.normal_()
    mods[1].load_state_dict(mods[0].state_dict())
    for m in mods:
        for name, p in m.named_parameters():
            p.requires_grad_(trained.get(name, True))
    return mods


@pytest.mark.parametrize("weight,bias,x", [(w, b, x) for w in (False, True) for b in (False, True) for x in (False, True)])
def test_any_of_the_inputs_may_be_the_one_that_is_trained(weight, bias, x):
    """A frozen weight beside a trained bias among them."""
    lib, ref = pair(48, weight=weight, bias=bias)
    t = torch.randn(6, 48, device=DEV)
    g = torch.randn_like(t)
    grads = []
    for m in (lib, ref):
        leaf = t.clone().requires_grad_(x)
        y = m(leaf)
        assert y.requires_grad == (weight or bias or x)
        if y.requires_grad:
            y.backward(g)
        grads.append((y.detach(), leaf.grad, m.weight.grad, m.bias.grad))
    for a, b in zip(*grads):
        assert (a is None) == (b is None)
        if a is not None:      # two fp32 orders of sums of 48 and of 6 terms
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)


def test_the_stem_trains_its_bias_alone():
    from dcnv4_b200.flash_intern_image import StemLayer
    torch.manual_seed(0)
    stem = StemLayer(3, 32, "GELU", "LN").to(DEV).requires_grad_(False)
    bias = stem.norm1[1].bias.requires_grad_(True)
    out = stem(torch.randn(2, 3, 32, 32, device=DEV))
    assert out.requires_grad
    out.square().sum().backward()
    assert bias.grad is not None and bias.grad.abs().sum() > 0


# ---- what only the stock operations support ------------------------------------------------------------------

def test_compiled_and_traced_modules():
    """One graph of stock operations, no break at the library's calls."""
    from dcnv4_b200.flash_intern_image import _post_norm, _pre_norm
    lib, ref = pair(24)
    t = torch.randn(6, 24, device=DEV)

    def block(m):
        def f(x):
            h, y = _pre_norm(m, x, x, torch.nn.Identity())
            return _post_norm(m, y, h, None, torch.nn.Identity()) + m(y)
        return f

    want = torch.autograd.grad(block(ref)(t.requires_grad_()).square().sum(), (t, ref.weight, ref.bias))
    got = torch.autograd.grad(torch.compile(block(lib), fullgraph=True, backend="eager")(t).square().sum(), (t, lib.weight, lib.bias))
    for a, b in zip(got, want):        # fp32 sums of 24 and 6 terms, three norms deep
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)
    from torch.fx.experimental.proxy_tensor import make_fx
    graph = make_fx(lambda x: lib(x), tracing_mode="real")(t.detach())
    assert any("layer_norm" in str(n.target) for n in graph.graph.nodes)
    other = torch.randn(6, 24, device=DEV)
    torch.testing.assert_close(graph(other), ref(other), rtol=1e-5, atol=1e-5)
    traced = torch.jit.trace(lib, (t.detach(),), check_trace=False)
    assert "layer_norm" in str(traced.inlined_graph)


def test_tensor_subclasses_keep_their_class():
    class Tagged(torch.Tensor):
        pass

    lib, ref = pair(24)
    x = torch.randn(5, 24, device=DEV)
    y = lib(x.as_subclass(Tagged).requires_grad_())
    assert type(y) is Tagged
    torch.testing.assert_close(y.as_subclass(torch.Tensor), ref(x), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("which", ["plain", "gelu", "post", "pre", "pre f16"])
def test_batched_gradients(which):
    """Several gradients through one backward pass at once (vectorised Jacobians), against one after the other."""
    from dcnv4_b200 import AddLayerNormFunction, LayerNormFunction, LayerNormResidualFunction
    g = torch.Generator(device=DEV).manual_seed(4)
    t = torch.float16 if which == "pre f16" else torch.float32
    x, r = (torch.randn(4, 3, 20, device=DEV, generator=g).to(t).requires_grad_() for _ in range(2))
    w, b, gamma = (torch.randn(20, device=DEV, generator=g).requires_grad_() for _ in range(3))
    s = torch.tensor([1.0, 0.0, 2.0, 1.0], device=DEV)
    leaves = (x, r, w, b)
    if which in ("plain", "gelu"):
        leaves = (x, w, b)
        outs = (LayerNormFunction.apply(x, w, b, 1e-6, "none" if which == "plain" else "gelu"),)
    elif which == "post":
        leaves = (x, r, w, b, gamma)
        outs = (LayerNormResidualFunction.apply(x, r, w, b, 1e-6, gamma, s),)
    else:
        outs = AddLayerNormFunction.apply(x, r, w, b, 1e-6, s)
    grads = [torch.randn(5, *o.shape, device=DEV, generator=g).to(o.dtype) for o in outs]
    got = torch.autograd.grad(outs, leaves, grads, is_grads_batched=True, retain_graph=True)
    for i in range(5):
        one = torch.autograd.grad(outs, leaves, [v[i] for v in grads], retain_graph=True)
        for a, e in zip(got, one):
            # fp32 sums of 20 and 12 terms either way; in fp16 one rounding of each result, 2^-11, on both sides
            torch.testing.assert_close(a[i], e, rtol=1e-4 if e.dtype == torch.float32 else 2.0 ** -10 + 1e-4, atol=1e-4)


# ---- memory layout -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("which", ["module", "post", "pre", "pre f16"])
def test_a_strided_input_is_copied_once(which):
    """One copy in the forward pass, none to ask whether the kernels apply, none in the backward pass."""
    from dcnv4_b200.flash_intern_image import _post_norm, _pre_norm
    lib, ref = pair(64)
    t = torch.float32
    if which == "pre f16":
        t = torch.float16
        lib, ref = lib.half(), ref.half()
    base = torch.randn(2, 64, 50, device=DEV, dtype=t)
    grads, copies = [], []
    for m in (lib, ref):
        leaf = base.clone().requires_grad_()
        x = leaf.transpose(1, 2)
        res = torch.randn(2, 50, 64, device=DEV, dtype=t, generator=torch.Generator(device=DEV).manual_seed(1))
        with torch.autograd.profiler.profile() as prof:
            if which == "module":
                out = (m(x),)
            elif which == "post":
                out = (_post_norm(m, x, res, None, torch.nn.Identity()),)
            else:
                out = _pre_norm(m, x, res, torch.nn.Identity())
            (g,) = torch.autograd.grad(out, leaf, [o.detach() for o in out])      # contiguous gradients
        copies.append(sum(e.name == "aten::clone" for e in prof.function_events))
        grads.append(g)
    assert copies[0] == 1
    # fp32: sums of 64 terms in two orders; fp16: roundings of out, of its gradient and of the stored sum, 2^-11 each,
    # against values up to a few
    tol = 1e-4 if t == torch.float32 else 8 * 2.0 ** -11
    torch.testing.assert_close(grads[0], grads[1], rtol=tol, atol=tol * float(grads[1].abs().max()))


def test_second_derivative_through_a_strided_input():
    lib, ref = pair(24)
    outs = []
    base = torch.randn(24, 7, device=DEV)
    for m in (lib, ref):
        leaf = base.clone().requires_grad_()
        (g,) = torch.autograd.grad((m(leaf.t()) ** 3).sum(), leaf, create_graph=True)
        outs.append(torch.autograd.grad((g ** 2).sum(), leaf)[0])
    torch.testing.assert_close(outs[0], outs[1], rtol=1e-3, atol=1e-3 * float(outs[1].abs().max()))


@pytest.mark.parametrize("which", ["post, residual alone", "pre, weight alone and h", "pre f16, weight alone and h", "pre f16, residual alone"])
def test_differentiable_gradients_of_some_inputs_only(which):
    """create_graph=True where the wanted gradient does not go through the norm."""
    from dcnv4_b200 import AddLayerNormFunction, LayerNormResidualFunction
    g = torch.Generator(device=DEV).manual_seed(8)
    t = torch.float16 if "f16" in which else torch.float32
    x, r = (torch.randn(4, 16, device=DEV, generator=g).to(t) for _ in range(2))
    w, b = (torch.randn(16, device=DEV, generator=g) for _ in range(2))
    v = torch.randn(4, 16, device=DEV, generator=g).to(t)
    leaf = (r if "residual" in which else w).requires_grad_()
    if which.startswith("post"):
        out = LayerNormResidualFunction.apply(x, r, w, b, 1e-6)
        (got,) = torch.autograd.grad(out, leaf, v, create_graph=True)
        assert torch.equal(got, v)
    elif "weight" in which:
        h, y = AddLayerNormFunction.apply(x, r, w, b, 1e-6)
        (got,) = torch.autograd.grad(h, leaf, v, create_graph=True, allow_unused=True)
        assert got is None or not got.any()
    else:
        h, y = AddLayerNormFunction.apply(x, r, w, b, 1e-6)
        (got,) = torch.autograd.grad(h, leaf, v, create_graph=True)
        assert torch.equal(got, v)
