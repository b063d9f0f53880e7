"""How far orthogonalised directions are from the formula in 64 bits before their
last rounding, against what ``ops.orthogonalize`` states: 1e-5 in the 2-norm.

A result of 16 bits is round(x), and x = want + e, so |got - want| is at most half
a step of the type there plus |e|: what is left of |got - want| beyond half a step is at
most |e|, whose 2-norm is the stated one (a step is taken at the larger of the two values,
which allows for a power of two between them)."""
import numpy as np
import pytest
import torch

from blitzgs_b200 import ops

pytestmark = pytest.mark.gpu

# significant bits, smallest exponent
FORMATS = {torch.float32: (24, -126), torch.bfloat16: (8, -126), torch.float16: (11, -14)}


def formula(u, steps=5, coefficients=ops.ORTHO_COEFFICIENTS, eps=1e-7):
    """The direction in 64 bits, from the definition; coefficients and eps as 32-bit numbers."""
    X = u.double()
    tall = X.shape[-2] > X.shape[-1]
    X = X.mT if tall else X
    a, b, c = (float(np.float32(v)) for v in coefficients)
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + float(np.float32(eps)))
    for _ in range(steps):
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.mT if tall else X


def beyond_rounding(got, want):
    """2-norm of what |got - want| exceeds half a step of got's type by, over want's."""
    bits, least = FORMATS[got.dtype]
    g = got.double()
    e = torch.frexp(torch.maximum(g.abs(), want.abs()))[1] - 1
    half = torch.exp2(e.clamp(min=least).double() - bits)
    return float(((g - want).abs() - half).clamp(min=0).norm() / want.norm())


def matrices(shape, dtype, device, seed=0):
    """A few strong directions over a floor of noise, as gradients of matrices are."""
    gen = torch.Generator().manual_seed(seed + sum(shape))
    k = max(1, min(shape[-2:]) // 16)
    low = torch.randn(*shape[:-1], k, generator=gen) @ torch.randn(*shape[:-2], k, shape[-1], generator=gen)
    return ((low / k ** 0.5 + 0.3 * torch.randn(shape, generator=gen)) * 1e-3).to(dtype).to(device)


@pytest.mark.parametrize("shape", [(24, 40), (64, 64), (128, 256), (7, 60, 33), (200, 1000), (300, 300), (1024, 1024),
                                   (1030, 1100), (2, 777, 201)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_directions_of_16_bits_are_exact_but_for_their_rounding(cuda_device, shape, dtype):
    g = matrices(shape, dtype, cuda_device)
    assert beyond_rounding(ops.orthogonalize(g), formula(g)) <= 1e-5


@pytest.mark.parametrize("shape", [(1, 3), (12, 3), (9, 14), (24, 40), (100, 250), (200, 150), (150, 160)])
def test_updates_far_smaller_than_eps(cuda_device, shape):
    """The direction is then small throughout (a^5 |u| / eps), and as exact."""
    base = matrices(shape, torch.float32, "cpu")
    for norm in (1e-9, 1e-10, 1e-12, 1e-14, 1e-17, 1e-25, 1e-33):
        g = (base * (norm / base.norm())).to(cuda_device)
        for steps in (1, 2, 5):
            got = ops.orthogonalize(g, steps=steps)
            assert beyond_rounding(got, formula(g, steps=steps)) <= 1e-5, (norm, steps)


@pytest.mark.parametrize("shape", [(9, 14), (24, 40), (100, 250), (200, 150), (150, 160)])
def test_many_steps_from_far_below_eps(cuda_device, shape):
    """Iterates that are small at first and not at last, and ones that shrink.  (1.875 is the largest
    factor of the convergent triple; every step is one of the same kind, and the roundings of early
    ones, 2^-22 each, are multiplied no more than the iterates themselves: the sum of 30 stays below
    30 * 4 * 2^-22 = 2.9e-5 of the result.)"""
    base = matrices(shape, torch.float32, "cpu")
    convergent, halving = (1.875, -1.25, 0.375), (0.5, 0.0, 0.0)
    for norm, steps, co in ((1e-12, 25, convergent), (1e-14, 30, convergent), (1e-17, 25, convergent),
                            (1e-25, 64, convergent), (1e-3, 30, halving), (1e-12, 30, halving)):
        g = (base * (norm / base.norm())).to(cuda_device)
        got, want = ops.orthogonalize(g, steps=steps, coefficients=co), formula(g, steps=steps, coefficients=co)
        assert float((got.double() - want).norm() / want.norm()) <= 30 * 4 * 2.0 ** -22, (norm, steps, co)


@pytest.mark.parametrize("shape", [(1, 3), (12, 3), (9, 14), (24, 40), (100, 250), (200, 150), (150, 160)])
def test_the_smallest_and_largest_updates_without_eps(cuda_device, shape):
    """The direction of what 32 bits hold, down to numbers that are denormal themselves."""
    base = matrices(shape, torch.float32, "cpu").double()
    for norm in (1e-20, 1e-30, 1e-34, 1e-37, 3e-39, 1e-41, 1e30, 1e38):
        g = (base * (norm / base.norm())).float().to(cuda_device)
        got = ops.orthogonalize(g, eps=0.0)
        assert beyond_rounding(got, formula(g, eps=0.0)) <= 1e-5, norm


# Of an error d in each operand of a product (two f16 terms: 2^-23 of X, A and B, and the low * low
# product left out, 2^-22: together 2^-22 in the mean), what arises in step k reaches the result
# multiplied by at most a^(5 - k) |X_k| / |X_5|.  For n of some hundred rows these factors are about
# 21, 21, 21, 20, 6 and 2; independent errors add up in squares, so to 43 * 2^-22 = 1e-5 if every
# direction is a weak one.  Summed without the registers' rounding, 1024 columns alone leave 4e-5.
STATED = 1e-5


@pytest.mark.parametrize("shape", [
    (1, 1), (1, 7), (2, 2), (15, 3), (4, 17), (3, 64), (4, 512), (4, 513), (9, 31), (16, 16), (16, 33), (50, 16, 16),
    (17, 17), (63, 64), (64, 65), (33, 200), (64, 700), (127, 129), (128, 128), (300, 70, 66), (128, 256), (129, 257),
    (200, 1000), (513, 130), (300, 300), (700, 640), (20, 150, 260), (40, 257, 130), (130, 5000), (1030, 1100),
    (1400, 1290), (1153, 2177), (2048, 1024), (3000, 3000), (2999, 3101)])
def test_32_bit_directions(cuda_device, shape):
    for seed in range(2):
        g = matrices(shape, torch.float32, cuda_device, seed)
        want = formula(g)
        assert float((ops.orthogonalize(g).double() - want).norm() / want.norm()) <= STATED


@pytest.mark.parametrize("shape", [(1, 1), (12, 3, 4), (100, 15, 3), (6, 16, 16), (20, 30), (3, 64, 64), (128, 256),
                                   (256, 128), (150, 200), (260, 200), (150, 201), (201, 150), (20, 150, 260),
                                   (7, 300, 130), (1400, 1292), (1292, 1400), (1401, 1291), (1291, 1401), (2048, 1024)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_updates(cuda_device, shape, dtype, nesterov):
    """Wide and tall, rows of whole fours of values and not, one tile to more than the grid has blocks:
    the momentum bit for bit, the parameter within the direction's stated error times lr scale and its
    own roundings (the two products' and the sum's, 2^-24 each of at most |param| + |step|)."""
    g = matrices(shape, dtype, cuda_device)
    M0, p0 = matrices(shape, torch.float32, cuda_device, 1), matrices(shape, torch.float32, cuda_device, 2) * 100
    p, M = p0.clone(), M0.clone()
    lr, beta, decay = 0.02, 0.95, 0.1
    ops.orthogonal_update(p, g, M, lr, beta=beta, nesterov=nesterov, weight_decay=decay)
    h = g.float() * (1 - beta)
    want_M = M0 * beta + h
    assert torch.equal(M, want_M)
    o = formula(h + want_M * beta if nesterov else want_M)
    alpha = lr * max(1.0, shape[-2] / shape[-1]) ** 0.5
    want = p0.double() * (1 - lr * decay) - alpha * o
    off, size = float((p.double() - want).norm()), float(p0.double().norm() + alpha * o.norm())
    assert off <= STATED * alpha * float(o.norm()) + 4 * 2.0 ** -24 * size
    assert not torch.equal(p, p0)
