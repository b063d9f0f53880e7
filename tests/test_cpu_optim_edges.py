"""CPU checks of the 8-bit optimizer state and the orthogonalised updates where they could go
wrong unnoticed: sizes past 32 bits and the wrappers' and optimizers' refusals."""
import pytest
import torch

from blitzgs_b200 import _lib, ops

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
