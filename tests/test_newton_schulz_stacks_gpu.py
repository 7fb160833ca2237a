"""Newton-Schulz in stacks: calls that follow one another without a pause."""
import pytest
import torch

from tests.test_newton_schulz_gpu import REL, check, few_rows, momentum, ref

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
