"""Orthogonalised matrices and the update along them, against the formula in 64 bits.

Tolerances (2-norm of the difference over the 2-norm of the result).  A
perturbation of relative size d of X before step k reaches the result
multiplied by at most a in each step left, so with |X_k|_F at most
min(a^k, 1.2 sqrt(n)) and the result's norm about 0.7 sqrt(n) or more,
    error <= d * sum_k a^(steps - k) min(a^k, 1.2 sqrt(n)) / (0.7 sqrt(n)) = d * G(n)
where a step's own roundings of A and B count like roundings of its X.  Two
f16 terms leave 2^-22 of each of X, A and B, and the low*low product that is left
out another 2^-22: d = 4 * 2^-22 = 2^-20.  In 32 bits (small matrices) d is smaller.
A bf16 result has its own half step (2^-9) and, from steps 3 and 4 computed
in one f16 term, at most 3 * 2^-12 (X, A, B rounded to nearest) times those two
steps' summands."""
import math

import numpy as np
import pytest
import torch

from blitzgs_b200 import _lib, ops
from oracle import optim_oracle as O

pytestmark = pytest.mark.gpu

A0 = ops.ORTHO_COEFFICIENTS[0]


def _gain(n, first=0, steps=5):
    return sum(A0 ** (steps - k) * min(A0 ** k, 1.2 * math.sqrt(n)) / (0.7 * math.sqrt(n))
               for k in range(first, steps + 1))


def _tol(n, dtype):
    t = 2.0 ** -20 * _gain(n)
    if dtype == torch.bfloat16:
        t += 2.0 ** -9 + 3 * 2.0 ** -12 * _gain(n, 3)
    elif dtype == torch.float16:
        t += 2.0 ** -12 + 2.0 ** -24 * math.sqrt(max(n, 1)) * 40  # and f16's smallest step on values near 1 / sqrt(m)
    return t


def _off(got, want):
    got = got.double().cpu().numpy()
    return np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300)


def _input(shape, dtype, seed=0, form="noise"):
    gen = torch.Generator().manual_seed(seed + sum(shape))
    g = torch.randn(shape, generator=gen)
    if form == "low":
        k = max(1, min(shape[-2:]) // 16)
        g = (torch.randn(*shape[:-1], k, generator=gen) @ torch.randn(*shape[:-2], k, shape[-1], generator=gen)
             + 0.1 * g)
    return (g * 1e-2).to(dtype)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 4), (15, 3), (4, 16), (4, 17), (3, 64), (2, 65), (4, 512), (4, 513),
          (5, 5), (9, 31), (16, 16), (16, 33), (17, 17), (63, 64), (33, 200), (64, 64), (65, 64), (64, 700), (65, 65),
          (127, 129), (128, 128), (129, 257), (200, 1000), (513, 130), (300, 300), (700, 640)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_matches_the_formula(cuda_device, shape, dtype):
    for form in ("noise", "low"):
        g = _input(shape, dtype, form=form)
        before = g.clone()
        got = ops.orthogonalize(g.to(cuda_device))
        assert got.dtype == dtype and got.shape == g.shape and torch.equal(g, before)
        assert _off(got, O.orthogonalize(g.double().numpy())) <= _tol(min(shape), dtype)


@pytest.mark.parametrize("shape", [(1030, 1100), (1400, 1290), (1153, 2177), (20, 150, 260), (40, 257, 130),
                                   (130, 5000), (3, 129, 385)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_many_tiles_and_long_sums(cuda_device, shape, dtype):
    """Sizes whose tiles are split over clusters or not, with odd numbers of tiles and of k blocks."""
    g = _input(shape, dtype, form="low")
    got = ops.orthogonalize(g.to(cuda_device))
    assert _off(got, O.orthogonalize(g.double().numpy())) <= _tol(min(shape[-2:]), dtype)


@pytest.mark.parametrize("shape", [(1000, 15, 3), (37, 3, 4), (50, 16, 16), (5, 40, 24), (7, 130, 70), (3, 2, 64, 200),
                                   (3, 300, 260), (200, 70, 66)])
def test_matrices_of_a_batch_do_not_touch_each_other(cuda_device, shape):
    g = _input(shape, torch.float32).to(cuda_device)
    flat = g.view(-1, *shape[-2:])
    flat[1] = 0
    flat[2, 0, 0] = float("nan")
    if flat.shape[0] > 4:
        flat[4, -1, -1] = float("inf")
    got = ops.orthogonalize(g).view(-1, *shape[-2:])
    assert (got[1] == 0).all() and got[2].isnan().all()
    if flat.shape[0] > 4:
        assert got[4].isnan().all()
    for b in (0, 3, flat.shape[0] - 1):
        if b < flat.shape[0] and b not in (1, 2, 4):
            assert _off(got[b], O.orthogonalize(flat[b].double().cpu().numpy())) <= _tol(min(shape[-2:]), torch.float32)


@pytest.mark.parametrize("shape", [(12, 3), (40, 60), (150, 130)])
def test_magnitudes(cuda_device, shape):
    """The direction does not depend on the update's size, from 1e-37 entries'
    squares to 1e30 ones', until eps matters."""
    base = _input(shape, torch.float32)
    for size in (1e-3, 1.0, 1e15, 1e32):
        got = ops.orthogonalize((base * size).to(cuda_device), eps=0.0)
        assert _off(got, O.orthogonalize((base * size).double().numpy(), eps=0.0)) <= _tol(min(shape), torch.float32)
    small = base * (1e-7 / base.norm())
    got = ops.orthogonalize(small.to(cuda_device), eps=1e-7)
    assert _off(got, O.orthogonalize(small.double().numpy(), eps=1e-7)) <= _tol(min(shape), torch.float32)


@pytest.mark.parametrize("shape", [(6, 4), (30, 50), (140, 100), (260, 300)])
def test_other_steps_and_coefficients(cuda_device, shape):
    """The cubic-convergent (15, -10, 3) / 8 drives every singular value to 1: after 25 steps the
    result is orthonormal, each entry of its Gram matrix to the products' 2^-20 a step (errors
    in converged directions are not multiplied: the polynomial's derivative there is 0)."""
    g = _input(shape, torch.float32)
    q = ops.orthogonalize(g.to(cuda_device), steps=25, coefficients=(1.875, -1.25, 0.375)).double().cpu()
    q = q if shape[0] <= shape[1] else q.t()
    gram = q @ q.t() - torch.eye(q.shape[0], dtype=torch.float64)
    assert gram.abs().max() <= 25 * 2.0 ** -20
    for steps in (1, 2):
        got = ops.orthogonalize(g.to(cuda_device), steps=steps)
        assert _off(got, O.orthogonalize(g.double().numpy(), steps=steps)) <= 2.0 ** -20 * _gain(min(shape))


def test_empty_and_strided(cuda_device):
    for shape in ((0, 4), (4, 0), (0, 3, 4), (3, 0, 0), (2, 0, 5)):
        assert ops.orthogonalize(torch.zeros(shape, device=cuda_device)).shape == shape
    g = _input((90, 160), torch.float32).to(cuda_device)
    for view in (g.t(), g[3:80, 5:150], g[::2, ::3], g[:, :1].expand(90, 160)[:, 1:]):
        assert torch.equal(ops.orthogonalize(view), ops.orthogonalize(view.clone().contiguous()))


@pytest.mark.parametrize("shape", [(500, 15, 3), (7, 9, 9), (5, 60, 100), (2, 150, 200)])
def test_entry_in_place_and_with_a_dirty_workspace(cuda_device, shape):
    """The C entry with out = g, and scratch full of NaN."""
    g = _input(shape, torch.float32).to(cuda_device)
    want = ops.orthogonalize(g)
    need = _lib.load().blitz_orthogonalize_workspace_bytes(*shape)
    ws = torch.full((need // 4 + 64,), float("nan"), device=cuda_device)
    _lib.call("blitz_orthogonalize", g.data_ptr(), 0, g.data_ptr(), *shape, 5, *ops.ORTHO_COEFFICIENTS, 1e-7,
              ws.data_ptr(), need, _lib.stream_ptr())
    torch.cuda.synchronize()
    assert torch.equal(g, want) and ws[need // 4:].isnan().all()


@pytest.mark.parametrize("shape", [(3, 4), (9, 9), (60, 100), (150, 200)])
def test_zeros_stay_zeros_without_eps(cuda_device, shape):
    assert (ops.orthogonalize(torch.zeros(shape, device=cuda_device), eps=0.0) == 0).all()


def test_more_small_matrices_than_a_grid_has_rows(cuda_device):
    """20 million 1 x 2 matrices.  A vector has one singular value, |g| / (|g| + eps) at
    first (eps shows in the shortest of so many), and the polynomial acts on it alone."""
    g = torch.randn(20_000_000, 1, 2, device=cuda_device)
    got = ops.orthogonalize(g).double().norm(dim=(1, 2))
    norm = g.double().norm(dim=(1, 2))
    s = norm / (norm + float(np.float32(1e-7)))
    for _ in range(5):
        a, b, c = (float(np.float32(v)) for v in ops.ORTHO_COEFFICIENTS)
        s = s * (a + b * s ** 2 + c * s ** 4)
    # 5 steps in 32 bits: each multiplies what came before by at most 3.45 and adds 6 roundings of 2^-24
    assert (got - s).abs().max() <= 6 * 2.0 ** -24 * sum(3.45 ** k for k in range(5)) + 1e-6


def test_a_repeated_call_gives_the_same_bits(cuda_device):
    for shape in ((15, 3), (50, 60), (300, 500), (4, 128, 256)):
        g = _input(shape, torch.float32).to(cuda_device)
        first = ops.orthogonalize(g)
        for _ in range(3):
            assert torch.equal(first, ops.orthogonalize(g))


def _update_reference(param, grad, momentum, lr, beta, nesterov, decay, scale):
    f = np.float32
    g, M = grad.float().numpy(), momentum.numpy()
    h = (g * f(1.0 - beta)).astype(f)
    M = ((M * f(beta)).astype(f) + h).astype(f)
    u = (h + (M * f(beta)).astype(f)).astype(f) if nesterov else M
    o = O.orthogonalize(u.astype(np.float64))
    return param.double().numpy() * (1 - lr * decay) - lr * scale * o, M, o


@pytest.mark.parametrize("shape", [(1, 1), (12, 3, 4), (100, 15, 3), (20, 30), (3, 64, 64), (128, 256), (300, 90), (2, 200, 130)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_update_matches_the_formula(cuda_device, shape, dtype, nesterov):
    """The momentum bit for bit; the parameter to the direction's tolerance times
    lr * scale, and two roundings of 2^-24."""
    grad, momentum, param = _input(shape, dtype), _input(shape, torch.float32, 1), _input(shape, torch.float32, 2) * 100
    p, M = param.to(cuda_device), momentum.to(cuda_device)
    lr, decay = 0.02, 0.1
    ops.orthogonal_update(p, grad.to(cuda_device), M, lr, nesterov=nesterov, weight_decay=decay)
    scale = math.sqrt(max(1.0, shape[-2] / shape[-1]))
    want, M_want, o = _update_reference(param, grad, momentum, lr, 0.95, nesterov, decay, scale)
    assert np.array_equal(M.cpu().numpy(), M_want)
    off = np.linalg.norm(p.cpu().double().numpy() - want)
    assert off <= lr * scale * _tol(min(shape[-2:]), torch.float32) * np.linalg.norm(o) \
        + 2 * 2.0 ** -24 * np.linalg.norm(want) + 2.0 ** -24 * lr * scale * np.linalg.norm(o)


def test_update_takes_a_given_scale_and_repeats(cuda_device):
    grad, param = _input((150, 200), torch.float32).to(cuda_device), torch.zeros(150, 200, device=cuda_device)
    M = torch.zeros_like(param)
    ops.orthogonal_update(param, grad, M, 0.5, beta=0.0, nesterov=False, scale=2.0)
    # param = -lr scale O: with lr scale = 1 the direction itself (beta 0: momentum = grad)
    assert torch.equal(M, grad) and torch.equal(param, -ops.orthogonalize(grad))


@pytest.mark.parametrize("shape", [(3, 15, 3), (60, 40), (200, 150)])
def test_on_other_streams_at_once_and_in_graphs(cuda_device, shape):
    """Calls in flight on two streams, and two captured graphs replayed in turn, each with its own scratch."""
    inputs = [_input(shape, torch.float32, s).to(cuda_device) for s in range(4)]
    want = [ops.orthogonalize(g) for g in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None] * 4
    for rounds in range(3):
        for k in range(4):
            with torch.cuda.stream(streams[k % 2]):
                got[k] = ops.orthogonalize(inputs[k])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graphs, outs, statics = [], [], [g.clone() for g in inputs[:2]]
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        streams[0].wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=streams[0]):
            outs.append(ops.orthogonalize(statics[k]))
        graphs.append(graph)
    for rounds in range(2):
        for k in range(2):
            statics[k].copy_(inputs[2 * rounds + k])
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(outs[k], want[2 * rounds + k])


def test_refusals(cuda_device):
    g = torch.zeros(5, 6, device=cuda_device)
    for bad, match in ((g.double(), "16 bits"), (g[0], "matrix"), (g.cpu(), "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            ops.orthogonalize(bad)
    for kw in (dict(steps=0), dict(steps=65), dict(coefficients=(10.0, -4.0, 2.0)), dict(eps=-1.0),
               dict(coefficients=(float("nan"), 0.0, 0.0)), dict(eps=float("nan"))):
        with pytest.raises(RuntimeError, match="blitz_orthogonalize"):
            ops.orthogonalize(g, **kw)
    with pytest.raises(RuntimeError, match="sizes"):
        ops.orthogonalize(torch.zeros(1, 40000, device=cuda_device))
    p, M = torch.zeros(5, 6, device=cuda_device), torch.zeros(5, 6, device=cuda_device)
    with pytest.raises(RuntimeError, match="different memory"):
        ops.orthogonal_update(p, g, p, 0.1)
    flat = torch.zeros(60, device=cuda_device)
    with pytest.raises(RuntimeError, match="different memory"):
        ops.orthogonal_update(flat[:30].view(5, 6), g, flat[20:50].view(5, 6), 0.1)
    ops.orthogonal_update(flat[:30].view(5, 6), g, flat[30:].view(5, 6), 0.1)
    with pytest.raises(RuntimeError, match="dense"):
        ops.orthogonal_update(p, g.to_sparse(), M, 0.1)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.orthogonal_update(p.t(), g.t(), M.t(), 0.1)
    with pytest.raises(RuntimeError, match="shape"):
        ops.orthogonal_update(p, g[:4], M, 0.1)
