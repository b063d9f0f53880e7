"""The 8-bit row store and the Adam step on it where they could go wrong unnoticed."""
import numpy as np
import pytest
import torch

from blitzgs_b200 import ops
from oracle import optim_oracle as O

pytestmark = pytest.mark.gpu

E4M3 = O.e4m3_values()


@pytest.mark.parametrize("D,group", [(256, 256), (48, 16), (20, 20), (255, 255), (51, 17), (6, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_every_byte_reads_as_the_format_has_it(cuda_device, D, group, dtype):
    """All 256 e4m3 bytes, the two NaN among them, and all int8 ones, at every kernel's widths,
    whole stores and listed rows."""
    n = -(-512 // D)
    raw = torch.arange(n * D, device=cuda_device).remainder(256).to(torch.uint8).view(n, D)
    scales = torch.exp2(torch.arange(n * -(-D // group), device=cuda_device).remainder(5).float() - 2).view(n, -1)
    size = scales.cpu().repeat_interleave(group, 1)[:, :D]
    for kind, number in ((torch.float8_e4m3fn, torch.from_numpy(E4M3)),
                         (torch.int8, torch.arange(256).to(torch.uint8).view(torch.int8).double())):
        want = (number[raw.cpu().long()] * size).to(dtype)
        for rows in (None, torch.arange(n - 1, -1, -1, device=cuda_device)):
            got = ops.quant_rows_read(raw.view(kind), scales, rows, group=group, dtype=dtype).cpu()
            assert torch.equal(got.isnan(), (want if rows is None else want.flip(0)).isnan())
            assert torch.equal(got.nan_to_num(7.0), (want if rows is None else want.flip(0)).nan_to_num(7.0))


def test_both_readers_of_a_nan_code_agree(cuda_device):
    """The Adam step takes the same bytes for NaN, in its element's parameter and its group's moments."""
    N, M = 4, 45
    codes = torch.full((N, M), 0x30, dtype=torch.uint8, device=cuda_device)
    codes[1, 7], codes[2, 44] = 0x7f, 0xff
    scales = torch.ones(N, 1, device=cuda_device)
    held = ops.quant_rows_read(codes.view(torch.float8_e4m3fn), scales, group=M)
    p = torch.zeros(N, M, device=cuda_device)
    root = torch.full((N, M), 0x30, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
    ops.adam8_update(p, torch.ones_like(p), codes.view(torch.float8_e4m3fn), scales, root, torch.ones_like(scales),
                     torch.ones(N, dtype=torch.bool, device=cuda_device), 0.1, 0.9, 0.999, 1e-15, N, M, group=M, seed=1)
    assert held.isnan().nonzero().tolist() == [[1, 7], [2, 44]]
    assert torch.equal(p.isnan(), held.isnan()) and scales.flatten().isnan().tolist() == [False, True, True, False]


def _rows(gen, n, M, spread):
    return torch.randn(n, M, generator=gen) * torch.exp(spread * torch.randn(n, 1, generator=gen))


@pytest.mark.parametrize("N,M,group", [(4000, 45, 128), (1000, 12, 12), (500, 100, 50), (200, 300, 256)])
@pytest.mark.parametrize("form", ["rows", "dense"])
def test_adam8_parameters_are_the_definitions_bit_for_bit(cuda_device, N, M, group, form):
    """Every operation of the step is rounded once, the quotient too: the parameter equals the
    restatement's in single float32 operations, as the 32-bit step's does."""
    gen = torch.Generator().manual_seed(M)
    param = torch.randn(N, M, generator=gen)
    p = param.to(cuda_device)
    stores = []
    for x in (_rows(gen, N, M, 1.0) * 1e-3, _rows(gen, N, M, 1.0).abs() * 1e-3):
        codes = torch.zeros((N, M), dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
        scales = torch.zeros((N, -(-M // group)), device=cuda_device)
        ops.quant_rows_write(x.to(cuda_device), codes, scales, group=group)
        stores += [codes, scales]
    m, r = (ops.quant_rows_read(*stores[k:k + 2], group=group).cpu().numpy() for k in (0, 2))
    grad = _rows(gen, N, M, 2.0) * 1e-3
    rows = torch.randperm(N, generator=gen)[:N // 2].sort().values
    if form == "rows":
        ops.adam8_update_rows(p, grad[rows].to(cuda_device), *stores, rows.to(cuda_device), 0.01, 0.9, 0.999, 1e-15, N, M,
                              group=group, seed=3)
    else:
        visible = torch.zeros(N, dtype=torch.bool)
        visible[rows] = True
        ops.adam8_update(p, grad.to(cuda_device), *stores, visible.to(cuda_device), 0.01, 0.9, 0.999, 1e-15, N, M,
                         group=group, seed=3)
    i = rows.numpy()
    want = param.numpy().copy()
    want[i] = O.adam8(want, grad.numpy()[i], m[i], r[i], i, 0.01, 0.9, 0.999, 1e-15, 3, group)[0]
    assert np.array_equal(p.cpu().numpy(), want)
