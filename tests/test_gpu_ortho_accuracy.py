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


@pytest.mark.parametrize("shape", [(1, 3), (12, 3), (9, 14), (24, 40), (100, 250), (200, 150), (150, 160)])
def test_the_smallest_and_largest_updates_without_eps(cuda_device, shape):
    """The direction of what 32 bits hold, down to numbers that are denormal themselves."""
    base = matrices(shape, torch.float32, "cpu").double()
    for norm in (1e-20, 1e-30, 1e-34, 1e-37, 3e-39, 1e-41, 1e30, 1e38):
        g = (base * (norm / base.norm())).float().to(cuda_device)
        got = ops.orthogonalize(g, eps=0.0)
        assert beyond_rounding(got, formula(g, eps=0.0)) <= 1e-5, norm
