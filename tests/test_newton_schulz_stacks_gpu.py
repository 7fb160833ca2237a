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


# ---- every form with every option ----------------------------------------------------------------------------

@pytest.mark.parametrize("batch,m,n", SIZES, ids=IDS)
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 10])
def test_steps_and_coefficients(batch, m, n, steps):
    """Results that end in either buffer, with and without steps that carry the pair, both iterations."""
    from dcnv4_b200 import ops
    x = momentum(batch, m, n)
    rel = REL * max(1, steps / 5)
    check(ops.newton_schulz(x, steps), ref(x, steps), rel)
    cubic = (1.5, -0.5, 0.0)
    check(ops.newton_schulz(x, steps, cubic), ref(x, steps, cubic), rel)
    assert ops.device_status() == 0


@pytest.mark.parametrize("batch,m,n", SIZES, ids=IDS)
def test_magnitudes_and_special_values(batch, m, n):
    from dcnv4_b200 import ops
    base = momentum(batch, m, n)
    for scale in (1e-3, 1e12, 1e25):
        check(ops.newton_schulz(base * scale), ref(base * scale))
    x = momentum(max(batch, 4), m, n)
    x[1] = 0
    x[2, 3, 5] = float("nan")
    y = ops.newton_schulz(x)
    assert not y[1].any() and y[2].isnan().all()
    keep = [i for i in range(len(x)) if i not in (1, 2)]
    check(y[keep], ref(x[keep]))
    x[2, 3, 5] = float("inf")
    y = ops.newton_schulz(x)
    assert not y[2].isfinite().any() and not y[1].any()
    check(y[keep], ref(x[keep]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("batch,m,n", SIZES + [(9, 1030, 1032)], ids=IDS + ["pairs of whole vectors"])
def test_unaligned_tensors(batch, m, n, dtype):
    """x one element into its storage, and an out that 16-byte stores cannot address, by the C entry point; the elements
    around out keep their values."""
    from dcnv4_b200 import _lib, ops
    x = momentum(batch, m, n, dtype)
    want = ops.newton_schulz(x)
    flat = torch.empty(x.numel() + 1, device=DEV, dtype=dtype)
    view = flat[1:].view(x.shape).copy_(x)
    assert torch.equal(ops.newton_schulz(view), want)
    L = _lib.lib()
    need = L.dcnv4b200_newton_schulz_workspace_bytes(batch, m, n)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    guard = torch.full((x.numel() + 130,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = guard[65:65 + x.numel()]
    a, b, c = ops.NEWTON_SCHULZ_COEFFICIENTS
    assert L.dcnv4b200_newton_schulz(x.data_ptr(), out.data_ptr(), ws.data_ptr(), need, {torch.float32: 0, torch.bfloat16: 2}[dtype],
                                     batch, m, n, 5, a, b, c, 1e-7, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out.view(x.shape), want)
    assert (guard[:65] == 7).all() and (guard[65 + x.numel():] == 7).all()


@pytest.mark.parametrize("m,n", [(1, 65536), (65536, 3), (40, 65535), (300, 65536), (129, 8)])
def test_long_and_thin(m, n):
    from dcnv4_b200 import ops
    from tests.test_newton_schulz_gpu import allowed
    x = momentum(1, m, n)
    check(ops.newton_schulz(x), ref(x), allowed(x))
    assert ops.device_status() == 0
