"""CPU checks of the 8-bit optimizer state and the orthogonalised updates: the
C ABI's argument checks (before any CUDA call), the wrappers' refusals, the
restatement against the format's definition, the optimizers' state handling with the
kernels replaced by the restatement, and its redistribution on gloo ranks."""
import ctypes
import os
import socket
import traceback

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from blitzgs_b200 import _lib, ops, optim
from blitzgs_b200 import redistribute as RD
from blitzgs_b200.rasterizer import SparseGaussianAdam
from oracle import optim_oracle as O

EINVAL, ESCRATCH = 10001, 10002


def _rejects(name, *args, code=EINVAL, msg=None):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    text = lib.blitz_last_error().decode()
    assert rc == code and name in text and (msg is None or msg in text), (name, rc, text)


def test_row_store_entries_check_their_arguments():
    w = "blitz_quant_rows_write"
    good = dict(values=16, type=0, stride=45, codes=16, scales=16, kind=1, rows=16, n=3, N=9, D=45, group=45, dither=0,
                seed=0, ptr=None, stream=None)

    def args(**kw):
        return list({**good, **kw}.values())

    for kw in (dict(n=-1), dict(N=-1), dict(D=-1), dict(D=2 ** 31), dict(group=0), dict(group=257), dict(kind=2),
               dict(type=3), dict(rows=None, n=10), dict(n=2 ** 60)):
        _rejects(w, *args(**kw), msg="bad sizes")
    _rejects(w, *args(stride=44), msg="value_stride")
    for kw in (dict(values=None), dict(codes=None), dict(scales=None)):
        _rejects(w, *args(**kw), msg="null pointer")
    assert _lib.call(w, *args(n=0, values=None)) == 0 and _lib.call(w, *args(D=0, values=None)) == 0
    r = "blitz_quant_rows_read"
    _rejects(r, 16, 16, 2, None, 3, 9, 45, 45, 16, 0, None, msg="bad sizes")
    _rejects(r, 16, 16, 1, None, 10, 9, 45, 45, 16, 0, None, msg="bad sizes")
    _rejects(r, 16, 16, 1, None, 3, 9, 45, 45, None, 0, None, msg="null pointer")
    _rejects(r, None, 16, 1, None, 3, 9, 45, 45, 16, 0, None, msg="null pointer")
    assert _lib.call(r, None, None, 0, None, 0, 0, 45, 45, None, 0, None) == 0


def test_adam8_entry_checks_its_arguments():
    a = "blitz_adam8_update"
    p = [16] * 6
    rest = [1.0, 0.1, 0.9, 0.1, 0.999, 0.001, 1e-15]
    _rejects(a, *p, 16, None, 0, *rest, -1, 45, 45, 0, None, None, msg="bad sizes")
    _rejects(a, *p, 16, None, 0, *rest, 5, 0, 45, 0, None, None, msg="bad sizes")
    _rejects(a, *p, 16, None, 0, *rest, 5, 45, 300, 0, None, None, msg="bad sizes")
    _rejects(a, *p, None, 16, -1, *rest, 5, 45, 45, 0, None, None, msg="bad sizes")
    _rejects(a, *p, 16, 16, 3, *rest, 5, 45, 45, 0, None, None, msg="either")
    _rejects(a, *p, None, None, 0, *rest, 5, 45, 45, 0, None, None, msg="either")
    for k in range(6):
        _rejects(a, *[None if i == k else 16 for i in range(6)], 16, None, 0, *rest, 5, 45, 45, 0, None, None,
                 msg="null pointer")
    assert _lib.call(a, *[None] * 6, None, 16, 0, *rest, 5, 45, 45, 0, None, None) == 0
    assert _lib.call(a, *[None] * 8, 0, *rest, 0, 45, 45, 0, None, None) == 0


def test_orthogonalisation_entries_check_their_arguments():
    co = [3.4445, -4.7750, 2.0315]

    def both(batch, rows, cols, steps=5, co=co, eps=1e-7, type=0, ptr=256, ws=256, size=2 ** 40, **kw):
        _rejects("blitz_orthogonalize", ptr, type, ptr, batch, rows, cols, steps, *co, eps, ws, size, None, **kw)
        _rejects("blitz_orthogonal_update", ptr, ptr, type, ptr, batch, rows, cols, steps, *co, eps, 0.95, 0.05, 1, 1.0,
                 0.1, ws, size, None, **kw)

    for sizes in ((-1, 4, 4), (1, -4, 4), (1, 4, 40000), (2 ** 40, 4, 4), (2 ** 24, 200, 200)):
        both(*sizes, msg="bad sizes")
    for kw in (dict(steps=0), dict(steps=65), dict(type=3), dict(eps=-1.0), dict(eps=float("nan"))):
        both(1, 300, 300, **kw, msg="bad sizes")
    for bad in ([8.0, -4.0, 1.0], [float("inf"), 0.0, 0.0], [float("nan"), 0.0, 0.0], [3.4445, -4.775, 9.0],
                [2.0, 0.0, 0.0]):
        both(1, 300, 300, co=bad, msg="coefficients")
    both(1, 300, 300, ptr=None, msg="null pointer")
    need = _lib.load().blitz_orthogonalize_workspace_bytes(1, 300, 300)
    assert need > 0
    both(1, 300, 300, size=need - 1, code=ESCRATCH, msg="workspace")
    both(1, 300, 300, ws=None, code=ESCRATCH, msg="workspace")
    both(1, 300, 300, ws=128, code=ESCRATCH, msg="workspace")
    for empty in ((0, 5, 5), (3, 0, 5), (3, 5, 0)):
        assert _lib.call("blitz_orthogonalize", None, 0, None, *empty, 5, *co, 1e-7, None, 0, None) == 0


def test_workspace_grows_with_the_batch_and_small_matrices_need_none():
    f = _lib.load().blitz_orthogonalize_workspace_bytes
    assert f(1000, 15, 3) == 0 and f(0, 300, 300) == 0 and f(1, 0, 300) == 0
    assert 0 < f(1, 300, 400) < f(2, 300, 400) and f(1, 300, 400) == f(1, 400, 300)


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(4, 45)
    codes, scales = torch.zeros(4, 45, dtype=torch.int8), torch.zeros(4, 1)
    f8 = torch.zeros(4, 45, dtype=torch.uint8).view(torch.float8_e4m3fn)
    for call in (lambda: ops.quant_rows_write(x, codes, scales, group=45),
                 lambda: ops.quant_rows_read(codes, scales, group=45),
                 lambda: ops.adam8_update(x, x, f8, scales, f8, scales, torch.ones(4).bool(), 0.1, 0.9, 0.999, 1e-15, 4,
                                          45, group=45, seed=0),
                 lambda: ops.orthogonalize(x), lambda: ops.orthogonal_update(x, x.clone(), x.clone(), 0.1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_restatement_rounds_to_the_nearest_value_of_the_format():
    """Against a search over every value that a byte can hold."""
    vals = np.unique(O.e4m3_values()[~np.isnan(O.e4m3_values())])
    x = np.random.default_rng(0).standard_normal((40, 45)).astype(np.float32) ** 5
    q, s = O.quantise(x, "e4m3", 45)
    y = x.astype(np.float64) / s
    assert np.isin(q, vals).all() and (np.abs(y).max(1) <= 448).all() and (np.abs(y).max(1) > 223).all()
    assert np.allclose(np.abs(q - y), np.abs(vals[None, None] - y[..., None]).min(-1), rtol=0, atol=0)
    u = O.row_uniforms(9, np.arange(40), 45)
    d, _ = O.quantise(x, "e4m3", 45, u)
    lo = vals[np.searchsorted(vals, np.abs(y), side="right") - 1]
    hi = vals[np.minimum(np.searchsorted(vals, np.abs(y), side="right"), len(vals) - 1)]
    assert ((np.abs(d) == lo) | (np.abs(d) == hi)).all()
    assert u.min() >= 0 and u.max() < 1 and abs(u.mean() - 0.5) < 0.05
    assert not np.array_equal(u, O.row_uniforms(10, np.arange(40), 45))
    big = O.row_uniforms(3, np.arange(2000), 50)
    # neighbouring rows, columns and seeds are uncorrelated: 1e5 pairs, five standard errors
    for a, b in ((big[:-1], big[1:]), (big[:, :-1], big[:, 1:]), (big, O.row_uniforms(4, np.arange(2000), 50)),
                 (big, O.row_uniforms(3 ^ O.ROOT_SALT, np.arange(2000), 50))):
        assert abs(np.corrcoef(a.ravel(), b.ravel())[0, 1]) < 5 / np.sqrt(a.size)


# ---------------------------------------------------------------------------
# the optimizers on the CPU, with the kernels replaced by their restatement
# ---------------------------------------------------------------------------

E4M3 = O.e4m3_values()


def _numbers(codes):
    return E4M3[codes.view(torch.uint8).numpy()].astype(np.float32)


def _bytes(q):
    """e4m3 numbers -> bytes."""
    vals = np.where(np.isnan(E4M3), np.inf, E4M3)
    order = np.argsort(vals, kind="stable")
    return torch.from_numpy(order[np.searchsorted(vals[order], q)].astype(np.uint8))


def _fake_adam8(param, grad, mc, ms, rc, rs, rows, lr, b1, b2, eps, N, M, *, group, seed, grad_scale=1.0):
    i = rows.numpy()
    p = param.detach().view(N, M)
    g = grad.detach().numpy().reshape(-1, M) * np.float32(grad_scale)
    m, r = (O.dequantise(_numbers(c)[i], s.numpy()[i], group) for c, s in ((mc, ms), (rc, rs)))
    out, (qm, sm), (qr, sr) = O.adam8(p.numpy(), g, m, r, i, lr, b1, b2, eps, seed, group)
    p[rows] = torch.from_numpy(out)
    for c, s, q, t in ((mc, ms, qm, sm), (rc, rs, qr, sr)):
        c.view(torch.uint8)[rows] = _bytes(q)
        s[rows] = torch.from_numpy(t)


@pytest.fixture
def fake_kernels(monkeypatch):
    monkeypatch.setattr(ops, "adam8_update_rows", _fake_adam8)
    monkeypatch.setattr(ops, "adam8_update", lambda param, grad, mc, ms, rc, rs, vis, *a, **k: _fake_adam8(
        param, grad.reshape(vis.numel(), -1)[vis], mc, ms, rc, rs, torch.nonzero(vis).flatten(), *a, **k))
    narrow = []
    monkeypatch.setattr(ops, "adam_update_rows", lambda *a, **k: narrow.append("rows"))
    return narrow


def test_sparse_adam_8bit_steps_and_state(fake_kernels):
    """Dense-with-mask and sparse gradients give the same state; rows of fewer than
    8 values take the 32-bit kernel; the direction follows the 32-bit Adam's."""
    gen = torch.Generator().manual_seed(0)
    N = 50
    base = torch.randn(N, 15, 3, generator=gen)
    opts, params = [], []
    for _ in range(2):
        p = torch.nn.Parameter(base.clone())
        q = torch.nn.Parameter(torch.zeros(N, 3))
        params.append((p, q))
        opts.append(optim.SparseGaussianAdam8bit([{"params": [p], "lr": 0.01}, {"params": [q], "lr": 0.01}], 0.0, 1e-15))
    assert isinstance(opts[0], SparseGaussianAdam)
    for t in range(3):
        vis = torch.rand(N, generator=gen) < 0.5
        g = torch.randn(N, 15, 3, generator=gen)
        rows = torch.nonzero(vis).flatten()
        for (p, q), opt, sparse in zip(params, opts, (False, True)):
            p.grad = torch.sparse_coo_tensor(rows[None], g[rows], (N, 15, 3)) if sparse else g.clone()
            q.grad = torch.sparse_coo_tensor(rows[None], g[rows, 0], (N, 3))
            opt.step(visibility=vis, N=N, bsz=4)
    a, b = (o.state[p[0]] for o, p in zip(opts, params))
    assert fake_kernels == ["rows"] * 6
    assert torch.equal(params[0][0], params[1][0])
    for k in ("exp_avg_codes", "exp_avg_scales", "exp_root_codes", "exp_root_scales"):
        assert torch.equal(a[k], b[k]) and a[k].shape[0] == N
    assert a["exp_avg_codes"].dtype == torch.uint8 and int(a["step"]) == 3
    # bytes of state a row: 2 * (45 + 4), against 360 in 32 bits
    assert sum(a[k].numel() * a[k].element_size() for k in a if k != "step") == N * 98
    # saving and loading keeps every byte, whatever the parameter's type does to a state tensor
    p2 = torch.nn.Parameter(base.clone())
    q2 = torch.nn.Parameter(torch.zeros(N, 3))
    opt2 = optim.SparseGaussianAdam8bit([{"params": [p2], "lr": 0.01}, {"params": [q2], "lr": 0.01}], 0.0, 1e-15)
    opt2.load_state_dict(opts[0].state_dict())
    for k in a:
        assert torch.equal(opt2.state[p2][k], a[k]) and opt2.state[p2][k].dtype == a[k].dtype
    # pruning and extending as the reference's model does with its moments
    keep = torch.arange(N) % 3 > 0
    assert torch.equal(a["exp_avg_codes"][keep], b["exp_avg_codes"][keep])
    grown = torch.cat((a["exp_root_codes"], torch.zeros(5, 45, dtype=torch.uint8)))
    assert (_numbers(grown)[N:] == 0).all()


def test_constructor_refusals():
    p = torch.nn.Parameter(torch.zeros(4, 45))
    with pytest.raises(ValueError, match="group"):
        optim.SparseGaussianAdam8bit([{"params": [p], "lr": 0.1}], 0.0, 1e-15, group=0)
    with pytest.raises(ValueError, match="matrices"):
        optim.OrthogonalMomentum([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="momentum_bits"):
        optim.OrthogonalMomentum([p], momentum_bits=4)
    with pytest.raises(ValueError, match="kind"):
        optim.QuantizedRows(4, 45, "cpu", kind="e5m2")
    with pytest.raises(ValueError, match="group"):
        optim.QuantizedRows(4, 45, "cpu", group=500)


def test_row_store_select_and_extend():
    st = optim.QuantizedRows(6, 5, "cpu", group=2)
    st.codes[:] = torch.arange(30).view(6, 5)
    st.scales[:] = torch.arange(18.0).view(6, 3)
    part = st.select(torch.tensor([4, 1]))
    assert torch.equal(part.codes, st.codes[[4, 1]]) and torch.equal(part.scales, st.scales[[4, 1]]) and len(part) == 2
    assert len(st.select(torch.arange(6) % 2 == 0)) == 3
    st.extend(2)
    assert len(st) == 8 and (st.codes[6:] == 0).all() and (st.scales[6:] == 0).all() and st.codes[5, 4] == 29


# ---------------------------------------------------------------------------
# redistribution
# ---------------------------------------------------------------------------

_SIZES = [70, 20]


def _worker(rank, ws, port, mode, q):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=ws)
    try:
        n = _SIZES[rank]
        g = torch.Generator().manual_seed(rank)
        ids = torch.arange(n) + 1000 * rank
        xyz = torch.nn.Parameter(torch.rand(n, 3, generator=g))
        feat = torch.nn.Parameter(ids[:, None].float().repeat(1, 9))
        opt = optim.SparseGaussianAdam8bit([{"params": [xyz], "lr": 0.1}, {"params": [feat], "lr": 0.1}], 0.0, 1e-15)
        opt.state[xyz] = {"step": torch.tensor(2.0), "exp_avg": xyz.detach() * 2, "exp_avg_sq": xyz.detach() * 3}
        opt.state[feat] = {"step": torch.tensor(2.0)}
        for j, k in enumerate(("exp_avg_codes", "exp_root_codes")):
            opt.state[feat][k] = ((ids[:, None] * 7 + torch.arange(9) + j) % 251).to(torch.uint8)
        for j, k in enumerate(("exp_avg_scales", "exp_root_scales")):
            opt.state[feat][k] = ids[:, None].float() * 0.5 + j
        new = RD.redistribute([xyz, feat], opt, mode=mode, force=True)
        st = opt.state[new[1]]
        ids = new[1].detach()[:, 0].long()
        ok = torch.equal(st["exp_avg_codes"], ((ids[:, None] * 7 + torch.arange(9)) % 251).to(torch.uint8))
        ok &= torch.equal(st["exp_root_codes"], ((ids[:, None] * 7 + torch.arange(9) + 1) % 251).to(torch.uint8))
        ok &= torch.equal(st["exp_avg_scales"], ids[:, None] * 0.5) and torch.equal(st["exp_root_scales"],
                                                                                    ids[:, None] * 0.5 + 1)
        ok &= torch.equal(opt.state[new[0]]["exp_avg"], new[0].detach() * 2)
        q.put((rank, ok, ids.tolist()))
    except Exception:
        q.put((rank, traceback.format_exc(), []))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("mode", ["round_robin", "zorder"])
def test_8bit_moments_travel_with_their_rows(mode):
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, mode, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = [q.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(60)
    assert all(g[1] is True for g in got), got
    assert sorted(got[0][2] + got[1][2]) == sorted(list(range(70)) + list(range(1000, 1020)))


def test_orthogonalisation_restatement_drives_singular_values_to_one():
    u = np.random.default_rng(1).standard_normal((2, 12, 30))
    s = np.linalg.svd(O.orthogonalize(u), compute_uv=False)
    assert ((s > 0.6) & (s < 1.25)).all()
    t = O.orthogonalize(np.swapaxes(u, 1, 2))
    assert np.allclose(np.swapaxes(t, 1, 2), O.orthogonalize(u), atol=1e-12)


def test_ctypes_pass_a_full_32_bit_seed():
    assert ctypes.c_int(0xFFFFFFFF).value == -1 and ops._seed(-1, None) == (0xFFFFFFFF, None)
