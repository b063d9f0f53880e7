"""The 8-bit row store and the sparse Adam step on it, against their numpy
restatement.  The store's arithmetic and the moments' are single float32 operations in
a fixed order, so codes and scales are compared bit for bit.  The parameter's step is a
quotient to 2 units in its last place: against the correctly rounded one, parameters
differ by at most 2^-22 of the step and one unit (2^-23) of the parameter."""
import numpy as np
import pytest
import torch

from blitzgs_b200 import ops
from oracle import optim_oracle as O

pytestmark = pytest.mark.gpu

KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
E4M3 = O.e4m3_values()


def _numbers(codes):
    """Stored bytes as the numbers they stand for before scaling (float32, numpy)."""
    b = codes.contiguous().view(torch.uint8).cpu().numpy()
    return (b.view(np.int8).astype(np.float32) if codes.dtype == torch.int8 else E4M3[b].astype(np.float32))


def _values(gen, n, D, spread=3.0):
    return torch.randn(n, D, generator=gen) * torch.exp(spread * torch.randn(n, 1, generator=gen))


def _store(N, D, group, kind, dev, fill=0):
    G = -(-D // group)
    codes = torch.full((N, D), fill, dtype=torch.uint8, device=dev).view(KINDS[kind])
    return codes, torch.full((N, G), float(fill), device=dev)


@pytest.mark.parametrize("D,group", [(1, 1), (1, 128), (3, 2), (8, 8), (9, 128), (16, 16), (17, 256), (45, 128),
                                     (64, 64), (65, 64), (128, 32), (200, 45), (256, 256), (257, 256), (1000, 67)])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("seed", [None, 12345])
def test_write_and_read_match_the_definition(cuda_device, D, group, kind, seed):
    gen = torch.Generator().manual_seed(D * 300 + group)
    N, n = 157, 61
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = _values(gen, n, D).clamp(-3e4, 3e4).to(dtype)
        x[3] = 0
        x[5, D // 2] = 0
        rows = torch.randperm(N, generator=gen)[:n]
        codes, scales = _store(N, D, group, kind, cuda_device, fill=5)
        ops.quant_rows_write(x.to(cuda_device), codes, scales, rows.to(cuda_device), group=group, seed=seed)
        u = None if seed is None else O.row_uniforms(seed, rows.numpy(), D)
        want, s = O.quantise(x.float().numpy(), kind, group, u)
        got = _numbers(codes)[rows.numpy()]
        assert np.array_equal(scales.cpu().numpy()[rows.numpy()], s)
        assert np.array_equal(got, want)
        # the stored value is within half a step (dithered: one) of the value, in 64 bits
        size = np.repeat(s.astype(np.float64), group, 1)[:, :D]
        step = size if kind == "int8" else np.maximum(2.0 ** -9 * size, np.abs(x.double().numpy()) * 2.0 ** -3)
        off = np.abs(got * size - x.double().numpy())
        # int8's quotient is rounded before it is made whole: at most 127 * 2^-24 < 2^-17 of a step more
        assert (off <= step * ((0.5 if seed is None else 1.0) + 2.0 ** -17)).all()
        # the other rows keep their bytes
        rest = np.setdiff1d(np.arange(N), rows.numpy())
        assert (codes.view(torch.uint8).cpu().numpy()[rest] == 5).all() and (scales.cpu().numpy()[rest] == 5).all()
        back = ops.quant_rows_read(codes, scales, rows.to(cuda_device), group=group)
        assert np.array_equal(back.cpu().numpy(), O.dequantise(want, s, group))
        for d in (torch.bfloat16, torch.float16):
            small = ops.quant_rows_read(codes, scales, rows.to(cuda_device), group=group, dtype=d)
            assert torch.equal(small.cpu(), torch.from_numpy(O.dequantise(want, s, group)).to(d))


def test_storing_stored_values_changes_nothing(cuda_device):
    gen = torch.Generator().manual_seed(3)
    x = _values(gen, 500, 45).to(cuda_device)
    codes, scales = _store(500, 45, 45, "e4m3", cuda_device)
    ops.quant_rows_write(x, codes, scales, group=45)
    first = ops.quant_rows_read(codes, scales, group=45)
    for seed in (None, 1, 2):
        ops.quant_rows_write(first, codes, scales, group=45, seed=seed)
        assert torch.equal(ops.quant_rows_read(codes, scales, group=45), first)


def test_extreme_values(cuda_device):
    D = 8
    tiny, huge = 1e-45, 3.4e38
    x = torch.zeros(10, D)
    x[0] = torch.tensor([huge, -huge, 1.0, 1e30, -1e37, 0.0, tiny, 2.0])
    x[1] = tiny
    x[2, 1] = float("nan")
    x[3, 2] = float("inf")
    x[4, 0] = float("-inf")
    x[5] = -0.0
    x[6] = 448.0
    x[7] = torch.tensor([448.0, 449.0, 447.9, 1.75, 1.76, 2.0 ** -9, 2.0 ** -10, 2.0 ** -11])
    x[8] = 2.0 ** -126
    x[9] = torch.finfo(torch.float32).max
    for kind in KINDS:
        for seed in (None, 7):
            codes, scales = _store(10, D, D, kind, cuda_device)
            ops.quant_rows_write(x.to(cuda_device), codes, scales, group=D, seed=seed)
            u = None if seed is None else O.row_uniforms(seed, np.arange(10), D)
            want, s = O.quantise(x.numpy(), kind, D, u)
            assert np.array_equal(scales.cpu().numpy(), s, equal_nan=True)
            assert np.array_equal(_numbers(codes), want)
            back = ops.quant_rows_read(codes, scales, group=D).cpu()
            # nothing non-finite is hidden, and it stays in its group
            assert back[2:5].isnan().all() and back[[0, 1, 5, 6, 7, 8, 9]].isfinite().all()


def test_rows_outside_the_store(cuda_device):
    N, D = 10, 45
    rows = torch.tensor([3, -1, 10, 2 ** 40, -2 ** 40, 9], device=cuda_device)
    x = torch.randn(6, D, device=cuda_device)
    codes, scales = _store(N, D, 45, "int8", cuda_device, fill=9)
    ops.quant_rows_write(x, codes, scales, rows, group=45)
    untouched = [r for r in range(N) if r not in (3, 9)]
    assert (codes.view(torch.uint8)[untouched] == 9).all() and (scales[untouched] == 9).all()
    back = ops.quant_rows_read(codes, scales, rows, group=45)
    assert (back[1:5] == 0).all()
    assert torch.equal(back[[0, 5]], ops.quant_rows_read(codes, scales, group=45)[[3, 9]])
    empty = torch.empty(0, dtype=torch.int64, device=cuda_device)
    ops.quant_rows_write(x[:0], codes, scales, empty, group=45)
    assert ops.quant_rows_read(codes, scales, empty, group=45).shape == (0, D)
    # int32 lists, and a store without rows or columns
    assert torch.equal(ops.quant_rows_read(codes, scales, rows[[0, 5]].int(), group=45), back[[0, 5]])
    for shape in ((0, 45), (5, 0)):
        c, s = _store(*shape, 45, "e4m3", cuda_device)
        ops.quant_rows_write(torch.empty(shape, device=cuda_device), c, s, group=45)
        assert ops.quant_rows_read(c, s, group=45).shape == shape


def test_values_with_strides_and_offsets(cuda_device):
    """Rows of a wider tensor, transposed and expanded values, stores that begin at odd addresses."""
    gen = torch.Generator().manual_seed(9)
    wide = _values(gen, 40, 61).to(cuda_device)
    for x in (wide[:, 7:30], wide.t()[5:28, :40].t(), wide[:1, 3:26].expand(40, 23), wide[::2, 1:24].repeat(2, 1)):
        a, b = _store(40, 23, 16, "e4m3", cuda_device), _store(40, 23, 16, "e4m3", cuda_device)
        ops.quant_rows_write(x, *a, group=16, seed=4)
        ops.quant_rows_write(x.clone().contiguous(), *b, group=16, seed=4)
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
    flat = torch.zeros(1 + 40 * 23, dtype=torch.uint8, device=cuda_device)
    odd = flat[1:].view(40, 23).view(torch.int8)
    scales = torch.zeros(1 + 40 * 2, device=cuda_device)[1:].view(40, 2)
    ops.quant_rows_write(wide[:, 1:24], odd, scales, group=16)
    want, s = O.quantise(wide[:, 1:24].cpu().numpy(), "int8", 16)
    assert np.array_equal(_numbers(odd), want) and np.array_equal(scales.cpu().numpy(), s)
    assert flat[0] == 0
    back = ops.quant_rows_read(odd, scales, group=16, dtype=torch.bfloat16)
    assert torch.equal(back.cpu(), torch.from_numpy(O.dequantise(want, s, 16)).bfloat16())


def test_offsets_past_32_bits(cuda_device):
    """A store of more than 2^32 values (4.5 GB)."""
    D, N = 256, (2 ** 32) // 256 + 5000
    codes = torch.zeros((N, D), dtype=torch.uint8, device=cuda_device).view(torch.int8)
    scales = torch.zeros((N, 1), device=cuda_device)
    rows = torch.tensor([0, 1, N // 2, 2 ** 24, N - 1], device=cuda_device)
    x = torch.randn(5, D, device=cuda_device)
    ops.quant_rows_write(x, codes, scales, rows, group=D)
    want, s = O.quantise(x.cpu().numpy(), "int8", D)
    assert np.array_equal(_numbers(codes[rows]), want)
    assert np.array_equal(ops.quant_rows_read(codes, scales, rows, group=D).cpu().numpy(), O.dequantise(want, s, D))
    assert int(scales.count_nonzero()) == 5


def test_dithering_keeps_the_mean(cuda_device):
    """Over many seeds the stored value averages to the value: K = 4096 seeds of
    a step-1 uniform dither have a standard error of at most step / 2 / sqrt(K)
    (a two-point distribution's deviation is at most half its spacing); six of
    those are allowed over 45 values."""
    x = torch.linspace(0.013, 1.0, 45, device=cuda_device).repeat(4, 1)
    total = torch.zeros(4, 45, dtype=torch.float64, device=cuda_device)
    K = 4096
    for seed in range(K):
        codes, scales = _store(4, 45, 45, "e4m3", cuda_device)
        ops.quant_rows_write(x, codes, scales, group=45, seed=seed)
        total += ops.quant_rows_read(codes, scales, group=45)
    step = torch.exp2(torch.floor(torch.log2(x.double())) - 3)
    assert ((total / K - x).abs() <= 6 * step / 2 / K ** 0.5).all()


def _moments(gen, N, M, group, dev):
    m = _values(gen, N, M, 1.0) * 1e-3
    r = _values(gen, N, M, 1.0).abs() * 1e-3
    r[7] = 0  # a row never updated
    m[7] = 0
    out = []
    for x in (m, r):
        codes, scales = _store(N, M, group, "e4m3", dev)
        ops.quant_rows_write(x.to(dev), codes, scales, group=group)
        out.append((codes, scales))
    return out


@pytest.mark.parametrize("N,M,group", [(300, 1, 128), (300, 3, 128), (200, 8, 8), (301, 45, 128), (100, 48, 45),
                                       (64, 100, 33), (33, 256, 256), (20, 700, 256)])
@pytest.mark.parametrize("form", ["rows", "dense"])
def test_adam8_matches_the_definition(cuda_device, N, M, group, form):
    """Three steps: parameters, codes and scales bit for bit."""
    gen = torch.Generator().manual_seed(N + M)
    dev = cuda_device
    (mc, ms), (rc, rs) = _moments(gen, N, M, group, dev)
    param = torch.randn(N, M, generator=gen)
    p = param.to(dev)
    ref = param.numpy().copy()
    m = [_numbers(mc), ms.cpu().numpy()]
    r = [_numbers(rc), rs.cpu().numpy()]
    for t in range(3):
        vis = torch.rand(N, generator=gen) < 0.6
        vis[7] = t > 0
        rows = torch.nonzero(vis).flatten()
        grad = _values(gen, N, M, 2.0) * 1e-3
        grad[rows[0]] = 0
        lr, eps = 0.01, 1e-15
        if form == "rows":
            order = torch.randperm(rows.numel(), generator=gen)
            ops.adam8_update_rows(p, grad[rows][order].to(dev), mc, ms, rc, rs, rows[order].to(dev), lr, 0.9, 0.999,
                                  eps, N, M, group=group, seed=100 + t, grad_scale=0.5)
        else:
            ops.adam8_update(p, grad.to(dev), mc, ms, rc, rs, vis.to(dev), lr, 0.9, 0.999, eps, N, M, group=group,
                             seed=100 + t, grad_scale=0.5)
        i = rows.numpy()
        g = grad.numpy()[i] * np.float32(0.5)
        want, (qm, sm), (qr, sr) = O.adam8(ref, g, O.dequantise(m[0][i], m[1][i], group),
                                           O.dequantise(r[0][i], r[1][i], group), i, lr, 0.9, 0.999, eps, 100 + t,
                                           group)
        got = p.cpu().numpy()
        assert (np.abs(got[i] - want) <= 2.0 ** -22 * np.abs(want - ref[i]) + 2.0 ** -23 * np.abs(want)).all()
        rest = np.setdiff1d(np.arange(N), i)
        assert np.array_equal(got[rest], ref[rest])
        ref, m[0][i], m[1][i], r[0][i], r[1][i] = got.copy(), qm, sm, qr, sr
        for got, s, w in ((mc, ms, m), (rc, rs, r)):
            assert np.array_equal(s.cpu().numpy(), w[1])
            assert np.array_equal(_numbers(got), w[0])
        # a root that has seen a gradient is never zero
        seen = np.repeat(r[1], group, 1)[:, :M][i] > 0
        assert (r[0][i][seen & (g != 0)] > 0).all()


def test_adam8_without_history_is_the_first_adam_step(cuda_device):
    """From zero moments: param - lr m / (r + eps) with m = 0.1 g, r = sqrt(0.001) |g|,
    whatever the store holds afterwards; three roundings of 2^-24 each side."""
    N, M = 50, 45
    gen = torch.Generator().manual_seed(1)
    grad, param = torch.randn(N, M, generator=gen), torch.zeros(N, M)
    p = param.to(cuda_device)
    m, r = _store(N, M, 128, "e4m3", cuda_device), _store(N, M, 128, "e4m3", cuda_device)
    ops.adam8_update(p, grad.to(cuda_device), *m, *r, torch.ones(N, dtype=torch.bool, device=cuda_device), 0.1, 0.9,
                     0.999, 1e-15, N, M, group=128, seed=1)
    g = grad.double()
    want = -0.1 * (0.1 * g) / (np.sqrt(0.001) * g.abs() + 1e-15)
    assert ((p.cpu().double() - want).abs() <= 8 * 2.0 ** -24 * want.abs() + 1e-12).all()


def test_adam8_non_finite_gradients_stay_in_their_row(cuda_device):
    N, M = 6, 45
    grad = torch.ones(N, M, device=cuda_device)
    grad[2, 5] = float("nan")
    grad[4, 0] = float("inf")
    p = torch.zeros(N, M, device=cuda_device)
    m, r = _store(N, M, 128, "e4m3", cuda_device), _store(N, M, 128, "e4m3", cuda_device)
    vis = torch.ones(N, dtype=torch.bool, device=cuda_device)
    ops.adam8_update(p, grad, *m, *r, vis, 0.1, 0.9, 0.999, 1e-15, N, M, group=128, seed=1)
    assert p[2, 5].isnan() and p[2, :5].isfinite().all() and p[[0, 1, 3, 5]].isfinite().all()
    assert m[1][[2, 4]].isnan().all() and m[1][[0, 1, 3, 5]].isfinite().all()


def test_adam8_rows_outside_are_skipped(cuda_device):
    N, M = 9, 12
    rows = torch.tensor([2, -1, 9, 2 ** 33, 8], device=cuda_device)
    p = torch.zeros(N, M, device=cuda_device)
    m, r = _store(N, M, 12, "e4m3", cuda_device), _store(N, M, 12, "e4m3", cuda_device)
    ops.adam8_update_rows(p, torch.ones(5, M, device=cuda_device), *m, *r, rows, 0.1, 0.9, 0.999, 1e-15, N, M, group=12,
                          seed=3)
    changed = p.abs().sum(1) > 0
    assert changed.nonzero().flatten().tolist() == [2, 8]
    assert (m[1] > 0).flatten().nonzero().flatten().tolist() == [2, 8]


def test_adam8_with_nothing_to_update(cuda_device):
    """An empty row list, a mask without a visible Gaussian, a scene without Gaussians."""
    N, M = 7, 45
    p = torch.randn(N, M, device=cuda_device)
    before = p.clone()
    m, r = _store(N, M, 45, "e4m3", cuda_device), _store(N, M, 45, "e4m3", cuda_device)
    args = (0.1, 0.9, 0.999, 1e-15)
    ops.adam8_update_rows(p, p[:0].clone(), *m, *r, torch.empty(0, dtype=torch.int64, device=cuda_device), *args, N, M,
                          group=45, seed=1)
    ops.adam8_update(p, torch.ones_like(p), *m, *r, torch.zeros(N, dtype=torch.bool, device=cuda_device), *args, N, M,
                     group=45, seed=1)
    assert torch.equal(p, before) and (m[1] == 0).all() and (r[1] == 0).all()
    m, r = _store(0, M, 45, "e4m3", cuda_device), _store(0, M, 45, "e4m3", cuda_device)
    ops.adam8_update(p[:0], p[:0].clone(), *m, *r, torch.zeros(0, dtype=torch.bool, device=cuda_device), *args, 0, M,
                     group=45, seed=1)


def test_adam8_in_a_captured_graph_takes_its_seed_from_the_device(cuda_device):
    """A seed tensor counted up between replays gives each its own dithering: the
    replayed steps equal eager ones with the same seeds."""
    N, M = 40, 45
    gen = torch.Generator().manual_seed(2)
    grad = _values(gen, N, M).to(cuda_device)
    vis = torch.ones(N, dtype=torch.bool, device=cuda_device)

    def fresh():
        return (torch.zeros(N, M, device=cuda_device), _store(N, M, 45, "e4m3", cuda_device),
                _store(N, M, 45, "e4m3", cuda_device))

    def step(s, seed):
        ops.adam8_update(s[0], grad, *s[1], *s[2], vis, 0.1, 0.9, 0.999, 1e-15, N, M, group=45, seed=seed)

    eager, graphed = fresh(), fresh()
    for t in range(1, 5):
        step(eager, t)
    counter = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        counter += 1
        step(graphed, counter)
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager[0], graphed[0])
    for a, b in zip((*eager[1], *eager[2]), (*graphed[1], *graphed[2])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals(cuda_device):
    dev = cuda_device
    codes, scales = _store(4, 45, 16, "int8", dev)
    x = torch.zeros(4, 45, device=dev)
    with pytest.raises(RuntimeError, match="group"):
        ops.quant_rows_write(x, codes, scales, group=257)
    with pytest.raises(RuntimeError, match="scales"):
        ops.quant_rows_write(x, codes, scales, group=45)
    with pytest.raises(RuntimeError, match="values"):
        ops.quant_rows_write(x.double(), codes, scales, group=16)
    with pytest.raises(RuntimeError, match="values"):
        ops.quant_rows_write(x[:3], codes, scales, group=16)
    with pytest.raises(RuntimeError, match="codes"):
        ops.quant_rows_read(codes.view(torch.uint8), scales, group=16)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.quant_rows_read(codes[:, :32], scales[:, :2], group=16)
    with pytest.raises(RuntimeError, match="rows"):
        ops.quant_rows_read(codes, scales, torch.zeros(2, 2, dtype=torch.int64, device=dev), group=16)
    with pytest.raises(RuntimeError, match="16 bits"):
        ops.quant_rows_read(codes, scales, group=16, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.quant_rows_write(x.cpu(), codes, scales, group=16)
    m, r = _store(4, 45, 16, "e4m3", dev), _store(4, 45, 16, "e4m3", dev)
    vis = torch.ones(4, dtype=torch.bool, device=dev)
    args = (0.1, 0.9, 0.999, 1e-15, 4, 45)
    with pytest.raises(RuntimeError, match="float8"):
        ops.adam8_update(x, x.clone(), codes, scales, *r, vis, *args, group=16, seed=0)
    with pytest.raises(RuntimeError, match="visible"):
        ops.adam8_update(x, x.clone(), *m, *r, vis[:3], *args, group=16, seed=0)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.adam8_update(x, x[:3].clone(), *m, *r, vis, *args, group=16, seed=0)
    with pytest.raises(RuntimeError, match="seed"):
        ops.adam8_update(x, x.clone(), *m, *r, vis, *args, group=16, seed=torch.zeros(2, dtype=torch.int64, device=dev))
