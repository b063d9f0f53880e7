"""The optimizers of blitzgs_b200.optim in uses that could go wrong unnoticed."""
import pytest
import torch

from blitzgs_b200 import ops, optim

pytestmark = pytest.mark.gpu


def _captures(step):
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        step()
    return graph


def test_steps_that_round_by_the_hosts_count_are_not_captured(cuda_device):
    """A replayed seed would round alike every time.  What is refused leaves no trace, and the
    next step outside of a capture is the first."""
    p, q = torch.nn.Parameter(torch.zeros(50, 45, device=cuda_device)), torch.nn.Parameter(
        torch.ones(20, 30, device=cuda_device))
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    visible = torch.ones(50, dtype=torch.bool, device=cuda_device)
    adam = optim.SparseGaussianAdam8bit([{"params": [p], "lr": 0.1}], 0.0, 1e-15)
    mat = optim.OrthogonalMomentum([q], momentum_bits=8)
    for step in (lambda: adam.step(visibility=visible, N=50), mat.step):
        with pytest.raises(RuntimeError, match="captured"):
            _captures(step)
        torch.cuda.synchronize()
    assert len(adam.state[p]) == 0 and len(mat.state[q]) == 0 and (p == 0).all() and (q == 1).all()
    adam.step(visibility=visible, N=50)
    mat.step()
    assert int(adam.state[p]["step"]) == 1 and (p < 0).all() and not (q == 1).all()


def test_a_captured_step_of_matrices_with_32_bit_momentum_repeats_the_eager_one(cuda_device):
    gen = torch.Generator().manual_seed(0)
    start, grad = torch.randn(3, 40, 60, generator=gen), torch.randn(3, 40, 60, generator=gen)
    params, opts = [], []
    for _ in range(2):
        params.append(torch.nn.Parameter(start.to(cuda_device)))
        params[-1].grad = grad.to(cuda_device)
        opts.append(optim.OrthogonalMomentum([params[-1]], lr=0.05))
        opts[-1].step()  # makes the state
    graph = _captures(opts[1].step)
    for _ in range(3):
        opts[0].step()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(params[0], params[1]) and torch.equal(*(o.state[p]["momentum_buffer"]
                                                               for o, p in zip(opts, params)))


@pytest.mark.parametrize("shape", [(777, 201), (1024, 1024), (2, 300, 260)])
def test_an_update_in_a_part_of_the_gpu_equals_one_on_the_whole(cuda_device, shape):
    """A context with 24 SMs takes fewer blocks of the kernel that needs all of its blocks at once.
    (The launch used to be refused there, after the momentum had been advanced.)"""
    from torch.cuda import green_contexts
    if not green_contexts.SUPPORTED:
        pytest.skip("torch was built without green contexts")
    gen = torch.Generator().manual_seed(0)
    param, grad, momentum = (torch.randn(shape, generator=gen).to(cuda_device) for _ in range(3))

    def update():
        p, M = param.clone(), momentum.clone()
        ops.orthogonal_update(p, grad, M, 0.1)
        torch.cuda.synchronize()
        return p, M

    want = update()
    part = green_contexts.GreenContext.create(num_sms=24, device_id=0)
    part.set_context()
    try:
        with torch.cuda.stream(part.Stream()):
            got = update()
    finally:
        part.pop_context()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(update(), want))


def test_rows_of_an_empty_store(cuda_device):
    codes = torch.zeros((0, 45), dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
    scales, rows = torch.zeros((0, 1), device=cuda_device), torch.tensor([0, 5, -1], device=cuda_device)
    x = torch.ones(3, 45, device=cuda_device)
    ops.quant_rows_write(x, codes, scales, rows, group=45)
    assert (ops.quant_rows_read(codes, scales, rows, group=45) == 0).all()
    ops.adam8_update_rows(torch.zeros(0, 45, device=cuda_device), x, codes, scales, codes.clone(), scales.clone(), rows,
                          0.1, 0.9, 0.999, 1e-15, 0, 45, group=45, seed=1)
