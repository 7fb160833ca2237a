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
