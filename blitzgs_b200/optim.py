"""Optimizers beside ``rasterizer.SparseGaussianAdam``, and the 8-bit row store
they keep their state in.

  * ``QuantizedRows``: rows of values in 8 bits with a scale per group, written
    and read by row (``ops.quant_rows_write`` / ``ops.quant_rows_read``);
  * ``SparseGaussianAdam8bit``: the sparse Adam with both moments in such
    rows: 2.2 bytes of state per SH coefficient instead of 8;
  * ``OrthogonalMomentum``: for parameters that are matrices (colour transforms
    per image, layers of a network trained beside the Gaussians), steps along
    the momentum with its singular values driven towards 1
    (``ops.orthogonal_update``); its momentum in 32 or in 8 bits.

The state is made of plain tensors with one row per row of the parameter, so
``state[key][mask]`` and ``torch.cat`` prune and extend it as the reference's
model does with its Adam moments (scene/gaussian_model.py), and
``redistribute`` moves it between ranks.
"""
import torch

from . import ops
from .rasterizer import SparseGaussianAdam

_KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _groups(D, group):
    return -(-D // group)


class QuantizedRows:
    """N rows of D values in 8 bits.

    ``kind``: "e4m3" (8-bit floats, the scale a power of two: every value keeps
    its relative precision, 2^-4, down to 2^-15 of its group's largest) or "int8"
    (steps of 1/127 of the group's largest).  ``group``: values that share a
    scale, 1 to 256 (a row is cut into ceil(D / group) groups).  ``codes`` is a
    uint8 [N, D] and ``scales`` a float32 [N, ceil(D / group)] tensor; a store
    begins as zeros."""

    def __init__(self, N, D, device, kind="e4m3", group=128):
        if kind not in _KINDS:
            raise ValueError(f"kind is 'e4m3' or 'int8', got {kind!r}")
        if not 1 <= group <= 256:
            raise ValueError(f"a group holds 1 to 256 values, got {group}")
        self.kind, self.group = kind, group
        self.codes = torch.zeros((N, D), dtype=torch.uint8, device=device)
        self.scales = torch.zeros((N, _groups(D, group)), dtype=torch.float32, device=device)

    def __len__(self):
        return self.codes.shape[0]

    def write(self, values, rows=None, seed=None):
        """Store values [n, D] at the rows (distinct; None: all rows).  ``seed``
        dithers the rounding, None rounds to nearest."""
        ops.quant_rows_write(values, self.codes.view(_KINDS[self.kind]), self.scales, rows, group=self.group,
                             seed=seed)

    def read(self, rows=None, dtype=torch.float32):
        """The rows' values [n, D] (None: all)."""
        return ops.quant_rows_read(self.codes.view(_KINDS[self.kind]), self.scales, rows, group=self.group,
                                   dtype=dtype)

    def select(self, index):
        """A store of the rows that a bool mask or an index list selects, in that order."""
        other = QuantizedRows(0, self.codes.shape[1], self.codes.device, self.kind, self.group)
        other.codes, other.scales = self.codes[index].contiguous(), self.scales[index].contiguous()
        return other

    def extend(self, n):
        """n more rows, zeros, behind the last."""
        self.codes = torch.cat((self.codes, self.codes.new_zeros((n, self.codes.shape[1]))))
        self.scales = torch.cat((self.scales, self.scales.new_zeros((n, self.scales.shape[1]))))


def _codes_back(state, keys):
    """Optimizer.load_state_dict casts every state tensor to the parameter's
    type; codes go back to the bytes they were (whole numbers, so exactly)."""
    for st in state.values():
        for k in keys:
            if k in st and st[k].dtype != torch.uint8:
                st[k] = st[k].to(torch.uint8)


def _not_captured(param, what):
    """A captured step would be replayed with one seed: rounded up or down at the same places every
    time, a moving average drifts from its values or stands still."""
    if param.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} takes its seed from the host's step count and cannot be captured into a graph: "
                           "capture the operators of ops with a seed tensor that the graph counts up")


class SparseGaussianAdam8bit(SparseGaussianAdam):
    """``SparseGaussianAdam`` with both moments in 8 bits: the same constructor,
    ``step(visibility, N, bsz)``, learning-rate correction, sparse gradients and
    rows left alone.  The step itself is computed in 32 bits; then the first
    moment and the root of the second are stored again as e4m3 with a
    power-of-two scale per ``group`` values of a row, rounded up or down at random (by a
    hash of the step, row and column, so a run repeats) because moving averages
    change by less than half a step of 8 bits at a time.

    Rows of fewer than 8 values keep 32-bit moments: a scale of 4 bytes a row
    would take back what the codes save.  A gradient that is not finite, or whose square
    is not, makes the moments of its whole group NaN (one scale holds them)."""

    _CODES = ("exp_avg_codes", "exp_root_codes")

    def __init__(self, params, lr, eps, group=128):
        super().__init__(params=params, lr=lr, eps=eps)
        if not 1 <= group <= 256:
            raise ValueError(f"a group holds 1 to 256 values, got {group}")
        self.values_per_scale = group
        # saved and loaded with the state that is laid out by it
        for g in self.param_groups:
            g["values_per_scale"] = group

    def _update(self, param, state, n, visibility, lr, eps, scale):
        M = param.numel() // n
        if M < 8:
            return super()._update(param, state, n, visibility, lr, eps, scale)
        _not_captured(param, "SparseGaussianAdam8bit")
        group = next((g.get("values_per_scale", self.values_per_scale) for g in self.param_groups
                      if g["params"][0] is param), self.values_per_scale)
        if len(state) == 0:
            state["step"] = torch.tensor(0.0, dtype=torch.float32)
            for k in ("exp_avg", "exp_root"):
                state[k + "_codes"] = torch.zeros((n, M), dtype=torch.uint8, device=param.device)
                state[k + "_scales"] = torch.zeros((n, _groups(M, group)), dtype=torch.float32, device=param.device)
        state["step"] += 1
        step = state["step"]
        lr_t = float(lr * (1 - 0.999 ** step) ** 0.5 / (1 - 0.9 ** step))
        moments = (state["exp_avg_codes"].view(torch.float8_e4m3fn), state["exp_avg_scales"],
                   state["exp_root_codes"].view(torch.float8_e4m3fn), state["exp_root_scales"])
        g = param.grad
        rest = dict(group=group, seed=int(step), grad_scale=1.0 if scale is None else scale)
        if g.is_sparse:
            g = g.coalesce()
            rows = g.indices()[0]
            ops.adam8_update_rows(param, g.values().reshape(rows.numel(), M), *moments, rows, lr_t, 0.9, 0.999, eps, n,
                                  M, **rest)
        else:
            ops.adam8_update(param, g, *moments, visibility, lr_t, 0.9, 0.999, eps, n, M, **rest)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        _codes_back(self.state, self._CODES)


class OrthogonalMomentum(torch.optim.Optimizer):
    """Steps of matrix parameters [..., rows, cols] along their orthogonalised
    momentum (``ops.orthogonal_update``); leading dimensions are a batch of
    matrices.  ``momentum_bits=8`` keeps the momentum as e4m3 rows, dithered."""

    def __init__(self, params, lr=0.02, beta=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=ops.ORTHO_COEFFICIENTS, eps=1e-7, momentum_bits=32):
        if momentum_bits not in (8, 32):
            raise ValueError(f"momentum_bits is 32 or 8, got {momentum_bits}")
        super().__init__(params, dict(lr=lr, beta=beta, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps, momentum_bits=momentum_bits))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() < 2:
                    raise ValueError(f"OrthogonalMomentum takes matrices, got a parameter {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    self._update(p, self.state[p], group)
        return loss

    def _update(self, p, state, group):
        how = dict(beta=group["beta"], nesterov=group["nesterov"], weight_decay=group["weight_decay"],
                   steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"])
        if group["momentum_bits"] == 32:
            if len(state) == 0:
                state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            ops.orthogonal_update(p, p.grad, state["momentum_buffer"], group["lr"], **how)
            return
        _not_captured(p, "OrthogonalMomentum with momentum_bits=8")
        rows, cols, values = p.numel() // p.shape[-1], p.shape[-1], min(p.shape[-1], 128)
        if len(state) == 0:
            state["step"] = torch.tensor(0.0, dtype=torch.float32)
            state["momentum_codes"] = torch.zeros((rows, cols), dtype=torch.uint8, device=p.device)
            state["momentum_scales"] = torch.zeros((rows, _groups(cols, values)), dtype=torch.float32,
                                                   device=p.device)
        state["step"] += 1
        codes = state["momentum_codes"].view(torch.float8_e4m3fn)
        momentum = ops.quant_rows_read(codes, state["momentum_scales"], group=values).view(p.shape)
        ops.orthogonal_update(p, p.grad, momentum, group["lr"], **how)
        ops.quant_rows_write(momentum.view(rows, cols), codes, state["momentum_scales"], group=values,
                             seed=int(state["step"]))

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        _codes_back(self.state, ("momentum_codes",))
