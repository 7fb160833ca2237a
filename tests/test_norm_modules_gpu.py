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
