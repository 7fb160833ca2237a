"""Newton-Schulz in stacks: calls that follow one another without a pause."""
import pytest
import torch

from tests.test_newton_schulz_gpu import DEV, REL, check, few_rows, momentum, ref

pytestmark = pytest.mark.gpu


def test_small_stacks_of_different_widths_back_to_back():
    """Blocks with different shares of tensor memory, more of them than the GPU holds, queued without waiting."""
    from dcnv4_b200 import ops
    xs = [momentum(400, m, n, torch.bfloat16) for m, n in ((32, 64), (128, 256), (64, 128), (16, 48), (96, 200))]
    want = [ops.newton_schulz(x) for x in xs]
    torch.cuda.synchronize()
    for _ in range(4):
        got = [ops.newton_schulz(x) for x in xs]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for x, y in zip(xs, want):
        check(y, ref(x), max(REL, few_rows(x)))       # the per-direction bound holds at any size
    assert ops.device_status() == 0


# ---- the lower end of fp16's range ---------------------------------------------------------------------------
# Sizes: one block per matrix, tiles by single blocks (wide and tall), tiles by pairs of blocks.
SIZES = [(2, 80, 120), (1, 128, 256), (2, 200, 328), (1, 328, 200), (9, 1030, 1025)]
IDS = ["small", "small full", "tiled", "tiled tall", "pairs"]


@pytest.mark.parametrize("batch,m,n", SIZES, ids=IDS)
@pytest.mark.parametrize("steps", [1, 2, 5, 10])
def test_norms_far_below_eps(batch, m, n, steps):
    """X_0 as small as |x| / eps: the same relative error as at |X_0| = 1.  The rounding bound counts fifteen roundings
    for five steps; more steps have more of them in proportion."""
    from dcnv4_b200 import ops
    x = momentum(batch, m, n)
    norm = float(x.flatten(1).norm(dim=1).max())
    for ratio in (1.0, 30.0, 1e3, 1e5, 1e8, 1e14, 1e20):
        check(ops.newton_schulz(x, steps, eps=norm * ratio), ref(x, steps, eps=norm * ratio), REL * max(1, steps / 5))
    for scale in (1e-10, 1e-16, 1e-30):                  # the default eps outweighs these
        y = x * scale
        check(ops.newton_schulz(y, steps), ref(y, steps), REL * max(1, steps / 5))
    assert ops.device_status() == 0


@pytest.mark.parametrize("batch,m,n", SIZES, ids=IDS)
def test_norms_at_the_ends_of_fp32(batch, m, n):
    """1 / (|x| + eps) beyond the normal fp32 numbers on either side."""
    from dcnv4_b200 import ops
    x = momentum(batch, m, n)
    x = x / x.abs().max()
    big = x * 2e38
    assert big.isfinite().all()
    check(ops.newton_schulz(big), ref(big))
    # subnormal inputs keep few bits of x, but are what they are: the reference reads the same values
    tiny = x * 1e-41
    assert tiny.any()
    check(ops.newton_schulz(tiny, eps=0.0), ref(tiny, eps=0.0))
    check(ops.newton_schulz(tiny, eps=1e-40), ref(tiny, eps=float(torch.tensor(1e-40))))


@pytest.mark.parametrize("batch,m,n", SIZES, ids=IDS)
def test_matrices_of_one_stack_have_ranges_of_their_own(batch, m, n):
    from dcnv4_b200 import ops
    x = momentum(4, m, n)
    scale = torch.tensor([1.0, 1e-12, 0.0, 1e-25], device=DEV).view(4, 1, 1)
    y = ops.newton_schulz(x * scale)
    keep = [0, 1, 3]
    check(y[keep], ref((x * scale)[keep]))
    assert not y[2].any()
    cubic = (1.5, -0.5, 0.0)
    check(ops.newton_schulz(x * scale, 12, cubic)[keep], ref((x * scale)[keep], 12, cubic), REL * 12 / 5)
