"""What the Muon optimiser refuses, without a GPU."""
import pytest
import torch

from dcnv4_b200.muon import Muon


def matrix(*shape, **kw):
    return torch.nn.Parameter(torch.zeros(*shape, **kw))


@pytest.mark.parametrize("group", [dict(params=[matrix(4)]), dict(params=[matrix(4, 4), torch.nn.Parameter(torch.tensor(1.0))]),
                                   dict(params=[matrix(4, 4)], lr=-1.0), dict(params=[matrix(4, 4)], momentum=1.0),
                                   dict(params=[matrix(4, 4)], ns_steps=101), dict(params=[matrix(4, 4)], adjust_lr="none"),
                                   dict(params=[matrix(4, 4)], ns_coefficients=(1.0, 2.0)),
                                   dict(params=[matrix(4, 4, dtype=torch.float64)]), dict(params=[matrix(65537, 1)]),
                                   dict(params=[matrix(1, 65537)])],
                         ids=["vector", "scalar", "lr", "momentum", "steps", "adjust", "coefficients", "float64", "tall", "wide"])
def test_groups_are_refused_whenever_they_come(group):
    """A vector in a later group would be orthogonalised as a column, that is, scaled to length one."""
    with pytest.raises(ValueError):
        Muon([group])
    opt = Muon([matrix(4, 4)])
    with pytest.raises(ValueError):
        opt.add_param_group(group)
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[matrix(6, 4)], ns_steps=3))
    assert len(opt.param_groups) == 2


def test_a_refused_step_changes_nothing():
    a, b = matrix(4, 4), matrix(4, 6)
    opt = Muon([dict(params=[a]), dict(params=[b])])
    a.grad = torch.ones(4, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        opt.step()
    b.grad = torch.ones(4, 6).to_sparse()
    with pytest.raises(RuntimeError):
        opt.step()
    assert not opt.state and not a.any()


def test_weights_too_large_for_muon_go_to_the_other_optimiser():
    from dcnv4_b200.muon import split_parameters
    model = torch.nn.Sequential(torch.nn.Linear(2, 65537, bias=False), torch.nn.Linear(4, 6))
    matrices, others = split_parameters(model)
    assert [tuple(p.shape) for p in matrices] == [(6, 4)]
    assert [tuple(p.shape) for p in others] == [(65537, 2), (6,)]
    Muon(matrices)
