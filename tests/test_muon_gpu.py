"""The Muon optimiser's state and what it refuses."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_momentum_is_kept_in_32_bits(t):
    """Under a constant gradient the momentum reaches it: 300 steps leave 0.95^300 = 2e-7 of the distance, and every step
    rounds by at most half a step of fp32, which the factor 0.05 a step sums up to 20 of them."""
    from dcnv4_b200 import Muon
    g = torch.Generator(device=DEV).manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(s, device=DEV, generator=g).to(t)) for s in ((24, 40), (24, 40), (16, 8, 3, 3))]
    ps[2].data = ps[2].data.contiguous(memory_format=torch.channels_last)
    opt = Muon(ps, lr=1e-3, momentum=0.95)
    for p in ps:
        p.grad = torch.randn(p.shape, device=DEV, generator=g).to(t)
    for _ in range(300):
        opt.step()
    for p in ps:
        m = opt.state[p]["momentum_buffer"]
        assert m.dtype == torch.float32 and m.stride() == p.grad.stride()
        assert bool(((m - p.grad.float()).abs() <= (2.1e-7 + 20 * 2.0 ** -24) * p.grad.float().abs()).all())
        assert p.dtype == t and torch.isfinite(p).all()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_loaded_state_goes_on_as_the_saved_one(t):
    from dcnv4_b200 import Muon
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.nn.Parameter(torch.randn(16, 24, device=DEV, generator=g).to(t))
    opt = Muon([w], lr=0.01)
    grads = [torch.randn(16, 24, device=DEV, generator=g).to(t) for _ in range(4)]
    for v in grads[:2]:
        w.grad = v
        opt.step()
    twin = torch.nn.Parameter(w.detach().clone())
    other = Muon([twin], lr=0.5)
    import copy
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for v in grads[2:]:
        w.grad, twin.grad = v, v.clone()
        opt.step()
        other.step()
        assert torch.equal(w, twin)
        assert torch.equal(opt.state[w]["momentum_buffer"], other.state[twin]["momentum_buffer"])
