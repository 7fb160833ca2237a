"""Newton-Schulz orthogonalisation against the iteration in 64 bits.

Tolerance.  The result is rounded to bf16: half a step, 2^-8 relative at most, 2^-8 / sqrt(3) in the 2-norm.  The
iteration: every fp16 rounding (of A, B, and of X in the last two steps) is relative 2^-11 at most, 2^-11 / sqrt(3) in
the 2-norm of the rounded matrix.  Five steps have fifteen of them; taken at full size and adding up they are
15 * 2^-11 / sqrt(3) = 4.2e-3, and with bf16's 2.3e-3 in quadrature 4.8e-3.  Single elements are held to eight times that
of the matrix' root mean square.

That counts on many independent roundings.  A matrix of a few rows has a few singular values only, and each rounding
of a diagonal entry of A or B moves one of them as a whole.  For those the bound is the first-order recursion of the
scalar iteration f(s) = a s + b s^3 + c s^5, step by step, with u = 2^-11 for every rounding at its worst:
    e <- |f'(s) s / f(s)| e + ( |b s^3 + 2 c s^5| u_A + |B| s u_B ) / |f(s)| + u_X
where u_A = 3 u while X is carried as a pair (A's rounding, and two of the 11-bit operand) and u after that, u_B = 2 u
and u likewise, and u_X = u where X itself is rounded.  At s = 1 (one row) that is 2.0e-2: the quintic's derivative
exceeds 1 there in places, so a single direction may amplify what an average over many does not.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
REL = 4.8e-3
A_, B_, C_ = 3.4445, -4.7750, 2.0315


def ref(x, steps=5, coef=(A_, B_, C_), eps=1e-7):
    a, b, c = coef
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        A = x @ x.mT
        x = a * x + (b * A + c * A @ A) @ x
    return x.mT if tall else x


def few_rows(x, steps=5, coef=(A_, B_, C_)):
    """The bound of the scalar recursion (see the module's text), over the singular values of one matrix or a stack."""
    a, b, c = coef
    u = 2.0 ** -11
    s = torch.linalg.svdvals(x.double())
    s = (s / s.square().sum(-1, keepdim=True).sqrt()).clamp_min(1e-12)
    e = torch.zeros_like(s)
    for k in range(steps):
        pair = k < steps - 2
        f = (a * s + b * s ** 3 + c * s ** 5).abs()
        B = (b * s ** 2 + c * s ** 4 + (0 if pair else a)).abs()
        e = ((a + 3 * b * s ** 2 + 5 * c * s ** 4) * s).abs() / f * e
        e = e + ((b * s ** 3 + 2 * c * s ** 5).abs() * (3 * u if pair else u) + B * s * (2 * u if pair else u)) / f
        e = e + (u if k + 1 >= steps - 2 else 0.0)
        s = f
    return float(e.max()) + 2.0 ** -8


def allowed(x):
    return REL if min(x.shape[-2:]) >= 16 else max(REL, few_rows(x))


def check(got, want, rel=REL):
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    d = (got.double() - want).flatten(0, -3) if want.dim() > 2 else (got.double() - want)[None]
    w = want.flatten(0, -3) if want.dim() > 2 else want[None]
    norm = w.flatten(1).norm(dim=1)
    off = d.flatten(1).norm(dim=1)
    assert bool((off <= rel * norm).all()), f"relative error {(off / norm).max().item():.3g}"
    rms = norm / math.sqrt(w[0].numel())
    worst = (d.abs().flatten(1) - 2.0 ** -8 * w.abs().flatten(1)).amax(1)
    assert bool((worst <= 8 * rel * rms).all()), f"element off by {(worst / rms).max().item():.3g} rms"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def momentum(batch, m, n, dtype=torch.float32, seed=0, noise=0.1):
    g = gen(seed + 7 * m + n)
    r = max(1, min(m, n) // 16)
    x = torch.randn(batch, m, r, device=DEV, generator=g) @ torch.randn(batch, r, n, device=DEV, generator=g) / r ** 0.5
    x = x + noise * torch.randn(batch, m, n, device=DEV, generator=g)
    return (x * 1e-3).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch,m,n", [(1, 64, 64), (3, 128, 128), (2, 64, 256), (2, 256, 64), (1, 160, 640), (1, 640, 160),
                                       (2, 200, 136), (3, 136, 200), (1, 272, 160), (1, 384, 520)])
def test_against_64_bits(batch, m, n, dtype):
    from dcnv4_b200 import ops
    x = momentum(batch, m, n, dtype)
    check(ops.newton_schulz(x), ref(x))
    assert ops.device_status() == 0


@pytest.mark.parametrize("m,n", [(1, 1), (1, 7), (7, 1), (3, 5), (17, 33), (33, 17), (65, 63), (129, 127), (127, 129), (100, 1001),
                                 (1001, 100), (257, 300), (31, 1440)])
def test_odd_sizes(m, n):
    from dcnv4_b200 import ops
    for dtype in (torch.float32, torch.bfloat16):
        x = momentum(2, m, n, dtype)
        check(ops.newton_schulz(x), ref(x), allowed(x))
    assert ops.device_status() == 0


@pytest.mark.parametrize("batch,m,n", [(40, 300, 260), (80, 130, 257), (150, 255, 333), (150, 333, 255), (40, 512, 264), (75, 257, 513),
                                       (12, 1000, 770), (9, 770, 1100), (6, 900, 1030), (8, 1031, 897), (9, 1030, 1025)])
def test_stacks_that_fill_the_gpu(batch, m, n):
    """Wide tiles, by one CTA and by pairs of them, with ragged rows and columns; both streams at once and captured."""
    from dcnv4_b200 import ops
    x = momentum(batch, m, n, torch.bfloat16)
    want = ops.newton_schulz(x)
    check(want, ref(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [ops.newton_schulz(x) for _ in range(2)]
    mine = [ops.newton_schulz(x) for _ in range(2)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in other + mine)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.newton_schulz(x)
    graph.replay()
    assert torch.equal(y, want)
    assert ops.device_status() == 0


def test_spectra():
    """Flat, decaying and nearly rank-deficient spectra: the pair (hi, lo) keeps the small directions."""
    from dcnv4_b200 import ops
    g = gen(5)
    m, n = 160, 640
    flat = torch.randn(m, n, device=DEV, generator=g)
    u = torch.linalg.qr(torch.randn(m, m, device=DEV, generator=g))[0]
    v = torch.linalg.qr(torch.randn(n, n, device=DEV, generator=g))[0][:m]
    decay = u @ torch.diag(1.0 / torch.arange(1, m + 1, device=DEV)) @ v
    thin = momentum(1, m, n, noise=0.01)[0]
    for x in (flat, decay, thin):
        check(ops.newton_schulz(x), ref(x))


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 10])
def test_steps_and_coefficients(steps):
    from dcnv4_b200 import ops
    x = momentum(1, 96, 160)
    check(ops.newton_schulz(x, steps), ref(x, steps), REL * max(1, steps / 5))
    cubic = (1.5, -0.5, 0.0)                              # the classical iteration: no A A term
    check(ops.newton_schulz(x, steps, cubic), ref(x, steps, cubic), REL * max(1, steps / 5))


def test_result_is_nearly_orthogonal():
    """Singular values end up in the band the quintic is made for, singular vectors stay."""
    from dcnv4_b200 import ops
    x = torch.randn(128, 320, device=DEV, generator=gen(1))
    y = ops.newton_schulz(x).double()
    s = torch.linalg.svdvals(y)
    assert 0.6 < s.min() and s.max() < 1.25
    u, _, vh = torch.linalg.svd(x.double(), full_matrices=False)
    core = u.T @ y @ vh.T
    assert (core - torch.diag(core.diagonal())).norm() < 2 * REL * core.norm()


def test_magnitudes_and_special_values():
    from dcnv4_b200 import ops
    base = momentum(1, 80, 120)
    for scale in (1e-3, 1.0, 1e12, 1e25):
        x = base * scale
        check(ops.newton_schulz(x), ref(x))
    x = momentum(4, 80, 120)
    x[1] = 0
    x[2, 3, 5] = float("nan")
    y = ops.newton_schulz(x)
    assert not y[1].any()
    assert y[2].isnan().all()
    check(y[[0, 3]], ref(x[[0, 3]]))
    assert torch.equal(y[0], ops.newton_schulz(x[0]))      # a matrix does not depend on its stack


def test_repeats_streams_and_graphs():
    from dcnv4_b200 import ops
    x = momentum(3, 200, 328)
    want = ops.newton_schulz(x)
    for _ in range(3):
        assert torch.equal(ops.newton_schulz(x), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [ops.newton_schulz(x) for _ in range(4)]
    mine = [ops.newton_schulz(x) for _ in range(4)]        # both streams at once, each with its own workspace
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in other + mine)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.newton_schulz(x)
    x.copy_(momentum(3, 200, 328, seed=9))
    graph.replay()
    assert torch.equal(y, ops.newton_schulz(x))


def test_unaligned_input_and_stacks():
    from dcnv4_b200 import ops
    x = momentum(2, 48, 72)
    flat = torch.empty(x.numel() + 1, device=DEV)
    view = flat[1:].view(x.shape).copy_(x)
    assert torch.equal(ops.newton_schulz(view), ops.newton_schulz(x))
    deep = x.view(2, 1, 48, 72)
    assert torch.equal(ops.newton_schulz(deep).view(2, 48, 72), ops.newton_schulz(x))
    assert ops.newton_schulz(x[:0]).shape == (0, 48, 72)


def test_refusals():
    from dcnv4_b200 import ops
    x = torch.randn(8, 16, device=DEV)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.newton_schulz(x.t())
    with pytest.raises(RuntimeError, match="matrix"):
        ops.newton_schulz(x[0])
    with pytest.raises(RuntimeError, match="float64|supports"):
        ops.newton_schulz(x.double())
    with pytest.raises(RuntimeError):
        ops.newton_schulz(x, 0)
    with pytest.raises(ValueError):
        ops.newton_schulz(x, 101)
