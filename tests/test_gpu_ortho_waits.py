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
