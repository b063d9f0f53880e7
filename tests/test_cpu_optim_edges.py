"""CPU checks of the 8-bit optimizer state and the orthogonalised updates where they could go
wrong unnoticed: sizes past 32 bits and the wrappers' and optimizers' refusals."""
import copy

import pytest
import torch

from blitzgs_b200 import _lib, ops, optim
from tests.test_cpu_optim import fake_kernels  # noqa: F401 (a fixture)

EINVAL = 10001


@pytest.mark.parametrize("M", [2 ** 30 + 1, 2 ** 31, 2 ** 31 + 45, 2 ** 33])
@pytest.mark.parametrize("rows", [None, 16])
def test_adam8_refuses_rows_whose_columns_pass_32_bits(M, rows):
    """The entry answers before it calls the GPU, as the row store's does for such a row."""
    lib = _lib.load()
    step = [1.0, 0.1, 0.9, 0.1, 0.999, 0.001, 1e-15]
    rc = lib.blitz_adam8_update(*[16] * 6, None if rows else 16, rows, 1 if rows else 0, *step, 1, M, 128, 0, None, None)
    assert rc == EINVAL and "bad sizes" in lib.blitz_last_error().decode()
    rc = lib.blitz_quant_rows_read(16, 16, 1, rows, 1, 1, M, 128, 16, 0, None)
    assert rc == EINVAL and "bad sizes" in lib.blitz_last_error().decode()


def test_what_has_no_backward_refuses_tensors_that_want_one():
    """Before anything else, so that no graph is cut unsaid; without gradients the calls go on
    (here as far as the refusal of CPU tensors)."""
    g = torch.zeros(4, 5, requires_grad=True)
    codes, scales = torch.zeros(4, 5, dtype=torch.int8), torch.zeros(4, 1, requires_grad=True)
    calls = (lambda: ops.orthogonalize(g), lambda: ops.orthogonalize(g * 2),
             lambda: ops.quant_rows_read(codes, scales, group=5))
    for call in calls:
        with pytest.raises(RuntimeError, match="backward"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.orthogonalize(g.detach())


@pytest.fixture
def no_kernels(monkeypatch):
    """The wrappers on CPU tensors, up to the calls of the library, which do nothing."""
    monkeypatch.setattr(ops, "_same_device", lambda *t: None)
    monkeypatch.setattr(ops, "ptr", lambda t: None)
    monkeypatch.setattr(_lib, "call", lambda *a: 0)
    monkeypatch.setattr(_lib, "stream_ptr", lambda: None)


def test_in_place_operators_raise_the_versions_of_what_they_write(no_kernels):
    """So that a backward pass through a parameter that has been stepped since is refused, as after
    torch's own optimizers, and no cache keyed by the version answers with what was there before."""
    N, M = 6, 45

    def store():
        return torch.zeros(N, M, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(N, 1)

    p, m, r, rows = torch.nn.Parameter(torch.ones(N, M)), store(), store(), torch.arange(N)
    args = (0.1, 0.9, 0.999, 1e-15, N, M)
    steps = {"adam8": lambda: ops.adam8_update(p, torch.ones(N, M), *m, *r, torch.ones(N).bool(), *args, group=M, seed=0),
             "rows": lambda: ops.adam8_update_rows(p, torch.ones(N, M), *m, *r, rows, *args, group=M, seed=0)}
    for step in steps.values():
        loss = (p * p).sum()
        before = [t._version for t in (p, *m, *r)]
        step()
        assert all(t._version > v for t, v in zip((p, *m, *r), before))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    w, M0 = torch.nn.Parameter(torch.ones(5, 6)), torch.zeros(5, 6)
    loss, before = (w * w).sum(), (w._version, M0._version)
    ops.orthogonal_update(w, torch.ones(5, 6), M0, 0.1)
    assert w._version > before[0] and M0._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    before = [t._version for t in m]
    ops.quant_rows_write(torch.ones(N, M), *m, group=M)
    assert all(t._version > v for t, v in zip(m, before))
    with torch.inference_mode():
        c, s = store()
        ops.quant_rows_write(torch.ones(N, M), c, s, group=M)


def _stepped(opt, p, grads):
    for g in grads:
        p.grad = g.clone()
        opt.step(visibility=torch.ones(p.shape[0]).bool(), N=p.shape[0])
    return p


@pytest.mark.parametrize("other", [64, 70, 128])
def test_a_loaded_state_keeps_the_groups_it_was_made_with(fake_kernels, other):  # noqa: F811
    """100 values in groups of 50 and of 64 have two scales each, but not of the same values: an
    optimizer made with other groups goes on with the loaded ones."""
    gen = torch.Generator().manual_seed(0)
    start, grads = torch.randn(6, 100, generator=gen), torch.randn(4, 6, 100, generator=gen)
    p, q = torch.nn.Parameter(start.clone()), torch.nn.Parameter(start.clone())
    first = optim.SparseGaussianAdam8bit([{"params": [p], "lr": 0.01}], 0.0, 1e-15, group=50)
    _stepped(first, p, grads[:2])
    with torch.no_grad():
        q.copy_(p)
    second = optim.SparseGaussianAdam8bit([{"params": [q], "lr": 0.01}], 0.0, 1e-15, group=other)
    # as a file would: torch itself loads tensors of the right type without copying them
    second.load_state_dict(copy.deepcopy(first.state_dict()))
    assert torch.equal(_stepped(first, p, grads[2:]), _stepped(second, q, grads[2:]))
    for k, t in first.state[p].items():
        assert torch.equal(t, second.state[q][k])


def test_groups_of_a_state_saved_without_their_size_are_the_optimizers(fake_kernels):  # noqa: F811
    """State that names no group size, and parameters added later."""
    p, q = torch.nn.Parameter(torch.zeros(6, 100)), torch.nn.Parameter(torch.zeros(6, 100))
    opt = optim.SparseGaussianAdam8bit([{"params": [p], "lr": 0.01}], 0.0, 1e-15, group=25)
    state = opt.state_dict()
    del state["param_groups"][0]["values_per_scale"]
    opt.load_state_dict(state)
    opt.add_param_group({"params": [q], "lr": 0.01})
    q.grad = torch.ones(6, 100)
    _stepped(opt, p, torch.ones(1, 6, 100))
    assert opt.state[p]["exp_avg_scales"].shape == opt.state[q]["exp_avg_scales"].shape == (6, 4)


def test_every_row_of_a_list_lies_outside_an_empty_store():
    """And is skipped, as documented: an empty tensor has no address, and needs none."""
    step = [1.0, 0.1, 0.9, 0.1, 0.999, 0.001, 1e-15]
    assert _lib.call("blitz_quant_rows_write", 16, 0, 45, None, None, 1, 16, 3, 0, 45, 45, 0, 0, None, None) == 0
    assert _lib.call("blitz_adam8_update", None, 16, *[None] * 4, None, 16, 3, *step, 0, 45, 45, 0, None, None) == 0
