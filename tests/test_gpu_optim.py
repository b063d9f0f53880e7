"""The optimizers of blitzgs_b200.optim as a trainer uses them: real gradients
of the fused step and of the rasterizer, several steps, every step checked
against the restatement in 64 bits (or bit for bit where it is single float32
operations)."""
import math

import numpy as np
import pytest
import torch

from blitzgs_b200 import ops, optim, rasterizer as RZ, scene as S, step as ST
from oracle import optim_oracle as O
from tests.helpers import activated, scene_params

pytestmark = pytest.mark.gpu

E4M3 = O.e4m3_values()


def _numbers(codes):
    return E4M3[codes.cpu().numpy()].astype(np.float32)


@pytest.mark.parametrize("sparse", [True, False])
def test_training_steps_with_8bit_moments(cuda_device, sparse):
    """Four steps of a small scene: SH coefficients through the 8-bit kernel, its state
    bit for bit the restatement's on the same gradient; the narrow parameters bit for
    bit SparseGaussianAdam's."""
    dev = cuda_device
    sc = S.tiny(seed=5, P=3000, H=96, W=128)
    params = [torch.nn.Parameter(t.clone()) for t in scene_params(sc, dev)]
    lrs = [1e-3, 5e-3, 1e-3, 5e-2, 2.5e-3, 1.25e-4]
    opt = optim.SparseGaussianAdam8bit([{"params": [p], "lr": lr} for p, lr in zip(params, lrs)], 0.0, 1e-15)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    plain = RZ.SparseGaussianAdam([{"params": [p], "lr": lr} for p, lr in zip(twins, lrs)], 0.0, 1e-15)
    N, rest = params[0].shape[0], params[5]
    state = None
    for t in range(4):
        cam = sc.cameras[t % len(sc.cameras)]
        gt = S.target_image(t, cam.image_height, cam.image_width).to(dev)
        rs = S.raster_settings(cam.to(dev), device=dev)
        opt.zero_grad(set_to_none=True)
        out = ST.view_loss(params, rs, gt, sparse_grad=sparse)
        out[0].backward()
        vis = out[3] > 0
        for p, q in zip(params, twins):
            q.data.copy_(p.data)
            q.grad = p.grad.clone()
        before = rest.detach().clone()
        g = rest.grad.to_dense() if sparse else rest.grad
        rows = torch.nonzero(vis).flatten()
        i = rows.cpu().numpy()
        g = g.reshape(N, 45)[rows].cpu().numpy()
        opt.step(visibility=vis, N=N, bsz=2)
        plain.step(visibility=vis, N=N, bsz=2)
        for p, q in list(zip(params, twins))[:5]:
            assert torch.equal(p, q)
        st = opt.state[rest]
        if state is None:
            state = [np.zeros((N, 45), np.float32), np.zeros((N, 1), np.float32)] * 2
            state = [x.copy() for x in state]
        lr = float(lrs[5] * (1 - 0.999 ** torch.tensor(t + 1.0)) ** 0.5 / (1 - 0.9 ** torch.tensor(t + 1.0)))
        m, r = O.dequantise(state[0][i], state[1][i], 128), O.dequantise(state[2][i], state[3][i], 128)
        want, (qm, sm), (qr, sr) = O.adam8(before.cpu().numpy().reshape(N, 45), g * np.float32(0.5), m, r, i, lr, 0.9,
                                           0.999, 1e-15, t + 1, 128)
        for k, x in enumerate((qm, sm, qr, sr)):
            state[k][i] = x
        ref, got = before.cpu().numpy().reshape(N, 45), rest.detach().cpu().numpy().reshape(N, 45)
        hidden = np.setdiff1d(np.arange(N), i)
        assert np.array_equal(got[hidden], ref[hidden])
        # the step's quotient is good to 2 units in its last place, the parameter rounded once
        assert (np.abs(got[i] - want) <= 2.0 ** -22 * np.abs(want - ref[i]) + 2.0 ** -23 * np.abs(want)).all()
        for k, key in enumerate(("exp_avg_codes", "exp_avg_scales", "exp_root_codes", "exp_root_scales")):
            got = _numbers(st[key]) if k % 2 == 0 else st[key].cpu().numpy()
            assert np.array_equal(got, state[k]), key
        assert len(i) > 0 and np.isfinite(got).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_colour_matrices_trained_beside_the_gaussians(cuda_device, bits):
    """Two optimizers as one trainer uses them: SH and geometry by the 8-bit sparse Adam, a
    3 x 4 colour matrix per image and a 96 x 160 layer by orthogonalised momentum, gradients through
    the full rasterizer.  Every step of the matrices against the formula in 64 bits."""
    dev = cuda_device
    sc = S.tiny(seed=6, P=2000, H=64, W=80)
    xyz, s, q, shs, o = (t.clone().requires_grad_(True) for t in activated(sc, dev))
    colour = torch.nn.Parameter(torch.eye(3, 4, device=dev).repeat(len(sc.cameras), 1, 1))
    gen = torch.Generator().manual_seed(0)
    layer = torch.nn.Parameter((torch.randn(96, 160, generator=gen) / 13).to(dev))
    adam = optim.SparseGaussianAdam8bit([{"params": [p], "lr": 1e-3} for p in (shs,)], 0.0, 1e-15)
    lr, decay = 0.02, 0.01
    ortho = optim.OrthogonalMomentum([colour, layer], lr=lr, weight_decay=decay, momentum_bits=bits)
    kept = {}
    for t in range(3):
        cam = sc.cameras[t % len(sc.cameras)].to(dev)
        rast = RZ.GaussianRasterizer(S.raster_settings(cam, device=dev))
        image, radii, _ = rast(xyz, torch.zeros_like(xyz), o, dc=shs[:, :1], shs=shs[:, 1:], scales=s, rotations=q)
        k = t % len(sc.cameras)
        mixed = torch.einsum("ij,jhw->ihw", colour[k][:, :3], image) + colour[k][:, 3, None, None]
        feat = torch.tanh(torch.nn.functional.adaptive_avg_pool2d(mixed, (10, 16)).reshape(3, 160) @ layer.t())
        gt = S.target_image(t, cam.image_height, cam.image_width).to(dev).float() / 255
        loss = (mixed - gt).abs().mean() + 0.1 * feat.square().mean()
        loss.backward()
        before = {p: p.detach().double().cpu().numpy() for p in (colour, layer)}
        grads = {p: p.grad.clone() for p in (colour, layer)}
        sh_before = shs.detach().clone()
        adam.step(visibility=radii > 0, N=shs.shape[0])
        ortho.step()
        assert torch.isfinite(shs).all() and not torch.equal(shs, sh_before)
        assert torch.equal(shs[radii == 0], sh_before[radii == 0])
        for p in (colour, layer):
            f, (rows, cols) = np.float32, p.shape[-2:]
            h = (grads[p].cpu().numpy() * f(1 - 0.95)).astype(f)
            M = kept.get(p, np.zeros(p.shape, f))
            M = ((M * f(0.95)).astype(f) + h).astype(f)
            u = (h + (M * f(0.95)).astype(f)).astype(f)
            # matrices whose image was not rendered have no momentum yet: zeros stay zeros
            scale = math.sqrt(max(1.0, rows / cols))
            want = before[p] * (1 - lr * decay) - lr * scale * O.orthogonalize(u.astype(np.float64))
            got = p.detach().double().cpu().numpy()
            # 5 steps multiply two f16 terms' 2^-20 by at most 485 and |X|'s growth (see test_gpu_ortho.py):
            # 4e-4 of |lr scale O| <= lr scale 1.2 sqrt(n), and the parameter's own roundings
            n = min(rows, cols)
            count = p.numel() // (rows * cols)
            assert np.linalg.norm(got - want) <= 4e-4 * lr * scale * 1.2 * math.sqrt(n * count) \
                + 3 * 2.0 ** -24 * np.linalg.norm(want)
            if bits == 32:
                kept[p] = M
                assert np.array_equal(ortho.state[p]["momentum_buffer"].cpu().numpy(), M)
            else:
                st = ortho.state[p]
                flat, grp = M.reshape(-1, cols), min(cols, 128)
                qm, sm = O.quantise(flat, "e4m3", grp, O.row_uniforms(t + 1, np.arange(flat.shape[0]), cols))
                assert np.array_equal(_numbers(st["momentum_codes"]), qm)
                assert np.array_equal(st["momentum_scales"].cpu().numpy(), sm)
                kept[p] = O.dequantise(qm, sm, grp).reshape(p.shape)
        for p in (xyz, s, q, shs, o, colour, layer):
            p.grad = None
    state = ortho.state_dict()
    again = optim.OrthogonalMomentum([torch.nn.Parameter(colour.detach().clone()),
                                      torch.nn.Parameter(layer.detach().clone())], momentum_bits=bits)
    again.load_state_dict(state)
    for a, b in zip(ortho.state.values(), again.state.values()):
        for k in a:
            assert torch.equal(a[k], b[k]) and a[k].dtype == b[k].dtype


def test_row_store_class(cuda_device):
    gen = torch.Generator().manual_seed(0)
    for kind in ("e4m3", "int8"):
        st = optim.QuantizedRows(100, 48, cuda_device, kind=kind, group=48)
        assert (st.read() == 0).all()
        x = torch.randn(30, 48, generator=gen)
        rows = torch.randperm(100, generator=gen)[:30]
        st.write(x.to(cuda_device), rows.to(cuda_device))
        want = O.dequantise(*O.quantise(x.numpy(), kind, 48), 48)
        assert np.array_equal(st.read(rows.to(cuda_device)).cpu().numpy(), want)
        keep = torch.zeros(100, dtype=torch.bool, device=cuda_device)
        keep[rows.to(cuda_device)] = True
        part = st.select(keep)
        assert torch.equal(part.read(), st.read()[keep])
        part.extend(3)
        assert len(part) == 33 and (part.read()[30:] == 0).all()


def test_matrix_optimizer_refuses_a_parameter_on_the_cpu(cuda_device):
    p = torch.nn.Parameter(torch.zeros(4, 5))
    p.grad = torch.ones(4, 5)
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.OrthogonalMomentum([p]).step()
    assert ops.ORTHO_COEFFICIENTS[0] == 3.4445
