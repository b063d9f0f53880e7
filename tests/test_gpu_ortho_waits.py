"""Orthogonalisation whose waits run out: the limit is set so low that some or all
of a call's ordinary waits exceed it.  Every one ends by itself, whatever the other waits do."""
import contextlib

import pytest
import torch

from blitzgs_b200 import _lib, ops

pytestmark = pytest.mark.gpu

SHAPES = [(20, 30), (64, 64), (3, 128, 256), (150, 200), (512, 512), (2, 300, 260), (777, 201), (1300, 1300)]
LIMITS = [0, 200, 1000, 3000, 10000]


@contextlib.contextmanager
def wait_limit(cycles):
    lib = _lib.load()
    before = lib.blitz_orthogonalize_wait_limit(cycles)
    try:
        yield before
    finally:
        lib.blitz_orthogonalize_wait_limit(before)


def _input(shape, device):
    gen = torch.Generator().manual_seed(sum(shape))
    return torch.randn(shape, generator=gen).to(device)


def test_the_limit_is_returned_and_put_back(cuda_device):
    with wait_limit(123) as before:
        assert before == 4_000_000_000
        assert _lib.load().blitz_orthogonalize_wait_limit(-1) == 123
    assert _lib.load().blitz_orthogonalize_wait_limit(-1) == before


@pytest.mark.parametrize("shape", SHAPES)
def test_calls_whose_waits_run_out_end_and_leave_the_next_one_alone(cuda_device, shape):
    g = _input(shape, cuda_device)
    want = ops.orthogonalize(g)
    for limit in LIMITS:
        with wait_limit(limit):
            ops.orthogonalize(g)
            torch.cuda.synchronize()
        assert torch.equal(ops.orthogonalize(g), want)


def _limits(call_is_right):
    """Limits to try: low ones, under which every block gives up at once, and many around the one from
    which a call ends rightly, where single blocks give up late."""
    edge = 500
    while edge < 10 ** 6:
        with wait_limit(edge):
            if call_is_right():
                break
        edge = edge * 5 // 4
    return LIMITS + [edge * k // 100 for k in range(40, 120)]


def _over_the_grid(shape):
    return min(shape[-2:]) > 128 or max(shape[-2:]) > 256


def _whole(got, want):
    """Which matrices were lost: every matrix is right to the last bit, or NaN throughout."""
    lost = got.flatten(1).isnan().all(1)
    assert torch.equal(got[~lost], want[~lost])
    return lost.tolist()


@pytest.mark.parametrize("shape", SHAPES)
def test_outputs_are_right_or_nan_throughout(cuda_device, shape):
    """Whichever block gives up, in whichever phase: nothing finite is left that is wrong.
    (The barriers of one block suspend a thread for longer than any of these waits lasts, so
    only waits over the grid run out.)"""
    g = _input(shape, cuda_device)
    flat = (-1,) + shape[-2:]
    want = ops.orthogonalize(g).view(flat)
    seen = set()
    for limit in _limits(lambda: torch.equal(ops.orthogonalize(g).view(flat), want)):
        with wait_limit(limit):
            lost = _whole(ops.orthogonalize(g).view(flat), want)
        if _over_the_grid(shape):
            assert len(set(lost)) == 1  # the call is lost as a whole
        seen.update(lost)
    assert True in seen or not _over_the_grid(shape)


@pytest.mark.parametrize("shape", [(3, 40, 60), (150, 200), (2, 300, 90), (700, 640)])
def test_updates_are_right_or_nan_throughout(cuda_device, shape):
    g, M0, p0 = (_input(shape, cuda_device) * k for k in (1.0, 0.5, 0.1))

    def update():
        p, M = p0.clone(), M0.clone()
        ops.orthogonal_update(p, g, M, 0.1, weight_decay=0.01)
        return p.view((-1,) + shape[-2:]), M

    want, M_want = update()
    seen = set()
    for limit in _limits(lambda: torch.equal(update()[0], want)):
        with wait_limit(limit):
            p, M = update()
            seen.update(_whole(p, want))
        assert torch.equal(M, M_want)
    assert True in seen or not _over_the_grid(shape)


@pytest.mark.parametrize("n", [300, 512, 768, 1024])
def test_a_block_that_gives_up_before_the_last_phase_is_not_lost_sight_of(cuda_device, n):
    """One step of a square 16-bit matrix: its first phase reads one term and the second two, so
    the longest wait, and the first to run out, is the one before the last phase."""
    g = _input((1, n, n), cuda_device).bfloat16()
    want = ops.orthogonalize(g, steps=1)
    for limit in _limits(lambda: torch.equal(ops.orthogonalize(g, steps=1), want)):
        with wait_limit(limit):
            for _ in range(3):
                _whole(ops.orthogonalize(g, steps=1), want)
