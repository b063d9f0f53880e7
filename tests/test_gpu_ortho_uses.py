"""Orthogonalisation as programs use it: several at once, beside other work, on tensors that
begin anywhere, on very long or very many matrices."""
import pytest
import torch

from blitzgs_b200 import ops
from tests.test_gpu_ortho_accuracy import STATED, beyond_rounding, formula, matrices

pytestmark = pytest.mark.gpu


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("shape", [(1, 4097), (1, 32768), (3, 20000), (2, 4, 5000), (16, 4097), (5, 30000), (32768, 3),
                                   (2, 9000, 17), (20, 32768)])
def test_long_matrices_with_few_rows(cuda_device, shape):
    for dtype in (torch.float32, torch.bfloat16):
        g = matrices(shape, dtype, cuda_device)
        assert beyond_rounding(ops.orthogonalize(g), formula(g)) <= STATED


def test_more_matrices_than_a_grid_has_rows(cuda_device):
    """65600 of 17 x 257, over the grid."""
    g = torch.randn(65600, 17, 257, device=cuda_device)
    got = ops.orthogonalize(g)
    for part in (slice(0, 100), slice(32768, 32800), slice(65500, 65600)):
        assert _off(got[part], formula(g[part])) <= STATED


@pytest.mark.parametrize("shape", [(500, 15, 3), (40, 4, 4), (30, 9, 12), (5, 64, 64), (2, 128, 256), (300, 260),
                                   (1030, 1100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_tensors_that_begin_anywhere(cuda_device, shape, dtype):
    """Contiguous, but one value past an aligned address: each of the three tensors in turn, and all."""
    def moved(t, by):
        flat = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
        flat[by:] = t.reshape(-1)
        return flat[by:].view(t.shape)

    g = matrices(shape, dtype, cuda_device)
    M0, p0 = matrices(shape, torch.float32, cuda_device, 1), matrices(shape, torch.float32, cuda_device, 2)
    assert beyond_rounding(ops.orthogonalize(moved(g, 1)), formula(g)) <= STATED
    p1, M1 = p0.clone(), M0.clone()
    ops.orthogonal_update(p1, g, M1, 0.1)
    for where in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        p, h, M = (moved(t, by) for t, by in zip((p0, g, M0), where))
        ops.orthogonal_update(p, h, M, 0.1)
        # the squares may be added up in another order (64 bits): the last bits of the direction
        assert torch.equal(M, M1) and _off(p, p1.double()) <= 2.0 ** -23


def test_calls_that_fill_the_gpu_on_several_streams_at_once(cuda_device):
    """Each needs all of its blocks at once, and gets them when the others are done; products of
    another stream run in between."""
    shapes = [(1024, 1024), (1300, 1300), (700, 640), (2000, 300)]
    inputs = [matrices(s, torch.float32, cuda_device, k) for k, s in enumerate(shapes)]
    want = [ops.orthogonalize(g) for g in inputs]
    big = torch.randn(4096, 4096, device=cuda_device)
    streams = [torch.cuda.Stream() for _ in range(5)]
    torch.cuda.synchronize()
    got = [[] for _ in shapes]
    for _ in range(15):
        with torch.cuda.stream(streams[4]):
            big = (big @ big).clamp_(-1, 1)
        for k, g in enumerate(inputs):
            with torch.cuda.stream(streams[k]):
                got[k].append(ops.orthogonalize(g))
    torch.cuda.synchronize()
    for k, w in enumerate(want):
        assert all(torch.equal(t, w) for t in got[k])


def test_graphs_that_fill_the_gpu_replayed_at_once(cuda_device):
    inputs = [matrices((900, 900), torch.float32, cuda_device, k) for k in range(2)]
    params = [torch.zeros(900, 900, device=cuda_device) for _ in range(2)]
    momenta = [torch.zeros(900, 900, device=cuda_device) for _ in range(2)]
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    for k in range(2):
        streams[k].wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graphs[k], stream=streams[k]):
            ops.orthogonal_update(params[k], inputs[k], momenta[k], 0.1)
    torch.cuda.synchronize()
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
    torch.cuda.synchronize()
    for k in range(2):
        p, M = torch.zeros_like(params[k]), torch.zeros_like(momenta[k])
        for _ in range(10):
            ops.orthogonal_update(p, inputs[k], M, 0.1)
        assert torch.equal(p, params[k]) and torch.equal(M, momenta[k])
