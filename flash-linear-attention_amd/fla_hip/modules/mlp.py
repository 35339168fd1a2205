"""The gated feed-forward block, with the interface of the reference's ``GatedMLP`` (fla/modules/mlp.py) and its three weights as one
differentiable function: ``y = (act(x Wg^T) * (x Wu^T)) Wd^T``.  All compute is done by ``gdn_gated_mlp_fwd`` and ``gdn_gated_mlp_bwd`` of the
HIP library, bf16 or fp16 operands with fp32 accumulators."""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from fla_hip import _lib
from fla_hip.ops.gated_delta_rule._common import aligned16, differentiable_once, dtype_code, launch, no_forward_mode, ptr, require_gpu, restored
from fla_hip.utils import calls_are_watched, calls_nothing_else

_ACTIVATIONS = {'swish': _lib.ACT_SILU, 'silu': _lib.ACT_SILU, 'sigmoid': _lib.ACT_SIGMOID, 'gelu_tanh': _lib.ACT_GELU_TANH}


def _pad(t: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """Contiguous, 16-byte aligned, with zeros up to ``rows x cols``."""
    r, c = rows - t.shape[0], cols - t.shape[1]
    return aligned16(F.pad(t, (0, c, 0, r)) if r or c else t.contiguous())


def _operands(x, gate_weight, up_weight, down_weight, keep):
    """The operands as the kernels read them: rows of a multiple of 8 elements."""
    M, D = x.shape
    if M <= _lib.MLP_FEW_ROWS and not keep:                                     # (a step of a few rows: of any width, at any address)
        return x.contiguous(), gate_weight.contiguous(), up_weight.contiguous(), down_weight.contiguous()
    D8, F8 = (D + 7) // 8 * 8, (gate_weight.shape[0] + 7) // 8 * 8
    return _pad(x, M, D8), _pad(gate_weight, F8, D8), _pad(up_weight, F8, D8), _pad(down_weight, D8, F8)


def _workspace(M, D, inner, backward, dev):
    n = _lib.load().gdn_gated_mlp_workspace_bytes(M, D, inner, backward)
    return (torch.empty(n, dtype=torch.uint8, device=dev) if n else None), n


def _forward(x, wg, wu, wd, activation, keep):
    M, D = x.shape
    inner = wg.shape[0]
    dev = x.device
    y = torch.empty_like(x)
    h = torch.empty(M, inner, dtype=x.dtype, device=dev)
    s, a = (torch.empty_like(h), torch.empty_like(h)) if keep else (None, None)
    ws, n = _workspace(M, D, inner, 0, dev)
    launch(_lib.load().gdn_gated_mlp_fwd, dev, ptr(x), ptr(wg), ptr(wu), ptr(wd), ptr(y), ptr(s), ptr(a), ptr(h), ptr(ws), n, M, D, inner,
           activation, dtype_code(x.dtype))
    return y, s, a, h


class GatedMLPFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, down_weight, activation):
        ops = _operands(x, gate_weight, up_weight, down_weight, True)
        need_x, need_g, need_u, need_d = ctx.needs_input_grad[:4]
        inner = need_x or need_g or need_u
        y, s, a, h = _forward(*ops, activation, inner)
        x_k, wg, wu, wd = ops
        ctx.save_for_backward(x_k if need_g or need_u else None, wg if need_x else None, wu if need_x else None, wd if inner else None,
                              s, a, h if need_d else None)
        ctx.sizes, ctx.kept = (*x.shape, gate_weight.shape[0]), (x.dtype, x.device)
        return y if y.shape == x.shape else y[:, :x.shape[1]].contiguous()

    @staticmethod
    @differentiable_once
    def backward(ctx, dy):
        need_x, need_g, need_u, need_d = ctx.needs_input_grad[:4]
        (M, D, inner), (dt, dev) = ctx.sizes, ctx.kept
        D8, F8 = (D + 7) // 8 * 8, (inner + 7) // 8 * 8
        shapes = ((M, D8), (F8, D8), (F8, D8), (D8, F8), *((M, F8),) * 3)
        x, wg, wu, wd, s, a, h = (restored(t, dt, shape, dev) for t, shape in zip(ctx.saved_tensors, shapes))
        dy = _pad(dy.to(device=dev, dtype=dt), M, D8)
        dg, du = (torch.empty_like(s), torch.empty_like(s)) if s is not None else (None, None)

        def empty(need, *shape):
            return torch.empty(shape, dtype=dt, device=dev) if need else None

        dx, dwg, dwu, dwd = empty(need_x, M, D8), empty(need_g, F8, D8), empty(need_u, F8, D8), empty(need_d, D8, F8)
        ws, n = _workspace(M, D8, F8, 1, dev)
        launch(_lib.load().gdn_gated_mlp_bwd, dev, ptr(dy), ptr(x), ptr(wg), ptr(wu), ptr(wd), ptr(s), ptr(a), ptr(h), ptr(dg), ptr(du),
               ptr(dx), ptr(dwg), ptr(dwu), ptr(dwd), ptr(ws), n, M, D8, F8, dtype_code(dt))

        def cut(t, rows, cols):
            return t if t is None or t.shape == (rows, cols) else t[:rows, :cols].contiguous()

        return cut(dx, M, D), cut(dwg, inner, D), cut(dwu, inner, D), cut(dwd, D, inner), None


def gated_mlp(
    x: torch.Tensor,
    gate_weight: torch.Tensor,
    up_weight: torch.Tensor,
    down_weight: torch.Tensor,
    activation: str = 'swish',
) -> torch.Tensor:
    """``(act(x @ gate_weight.T) * (x @ up_weight.T)) @ down_weight.T`` with ``x`` ``[..., D]``, ``gate_weight`` and ``up_weight`` ``[F, D]``,
    ``down_weight`` ``[D, F]``, all bf16 or all fp16; ``activation``: 'swish' / 'silu', 'sigmoid' or 'gelu_tanh'.  Differentiable in all four.
    Sums, activation and product are in fp32; the inner activation, what is kept for the backward and the inner gradients are rounded to the operands' type once each.
    Under autocast the operands are cast to its type first.  Without gradients up to 16 rows are read where they are, D and F of any
    size; otherwise D and F that are no multiples of 8 are zero-padded (copies of the weights per call)."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f'Unsupported activation: {activation}')
    if not torch.is_autocast_enabled():
        y = _lib.host().gated_mlp(x, gate_weight, up_weight, down_weight, _ACTIVATIONS[activation])
        if y is not None:
            return y
    if gate_weight.dim() != 2 or x.dim() < 1 or gate_weight.shape[1] != x.shape[-1]:
        raise ValueError(f'gate_weight must be [F, {x.shape[-1] if x.dim() else 1}] as x is {tuple(x.shape)}, got {tuple(gate_weight.shape)}')
    if up_weight.shape != gate_weight.shape or down_weight.shape != gate_weight.shape[::-1]:
        raise ValueError(f'up_weight must be shaped as gate_weight {tuple(gate_weight.shape)} and down_weight the other way round, '
                         f'got {tuple(up_weight.shape)} and {tuple(down_weight.shape)}')
    if 0 in gate_weight.shape:
        raise ValueError(f'the weights hold nothing: {tuple(gate_weight.shape)}')
    require_gpu(x, gate_weight, up_weight, down_weight)
    no_forward_mode('gated_mlp', x, gate_weight, up_weight, down_weight)
    if torch.is_autocast_enabled():
        x, gate_weight, up_weight, down_weight = (t.to(torch.get_autocast_dtype('cuda')) for t in (x, gate_weight, up_weight, down_weight))
    if any(w.dtype != x.dtype for w in (gate_weight, up_weight, down_weight)):
        raise ValueError(f'x and the weights must be of one dtype, got {x.dtype}, {gate_weight.dtype}, {up_weight.dtype}, {down_weight.dtype}')
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f'gated_mlp takes bf16 or fp16 operands, got {x.dtype}')
    x2 = x.reshape(-1, x.shape[-1])
    code = _ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, gate_weight, up_weight, down_weight)):
        y = GatedMLPFunction.apply(x2, gate_weight, up_weight, down_weight, code)
    else:
        y = _forward(*_operands(x2, gate_weight, up_weight, down_weight, False), code, False)[0]
        if y.shape != x2.shape:
            y = y[:, :x2.shape[1]].contiguous()
    return y.reshape(x.shape)


def _calls() -> tuple:
    return nn.Module.__call__, F.linear, nn.Linear.forward


# The calls that the operator stands for.  Where a caller has replaced one of them - here, on a module or around every module - the
# block runs projection by projection and makes it.
_CALLS = _calls()


class GatedMLP(nn.Module):
    """The feed-forward block as the reference's layer of that name builds it: no biases, the inner width ``hidden_ratio`` times two thirds of the hidden
    size, rounded up to a multiple of 256, unless it is given.  ``fuse_swiglu`` is taken for the reference's sake: there is one path.  That path is
    ``gated_mlp`` on the three weights, as long as calling the projections would do nothing else; adapters in their places, biases, hooks and the like are
    called, with the activation and the product in fp32 torch between them."""

    def __init__(
        self,
        hidden_size: int,
        hidden_ratio: int | None = None,
        intermediate_size: int | None = None,
        hidden_act: str = 'swish',
        fuse_swiglu: bool = True,
        device=None,
        dtype=None,
    ):
        super().__init__()
        if hidden_act not in _ACTIVATIONS:
            raise ValueError(f'Unsupported hidden_act: {hidden_act}')
        self.hidden_size = hidden_size
        if hidden_ratio is None:
            hidden_ratio = 4
        if intermediate_size is None:
            intermediate_size = int(hidden_size * hidden_ratio * 2 / 3)
            intermediate_size = 256 * ((intermediate_size + 256 - 1) // 256)
        self.hidden_ratio, self.intermediate_size, self.hidden_act, self.fuse_swiglu = hidden_ratio, intermediate_size, hidden_act, fuse_swiglu
        kwargs = {'device': device, 'dtype': dtype}
        self.gate_proj = nn.Linear(hidden_size, intermediate_size, bias=False, **kwargs)
        self.up_proj = nn.Linear(hidden_size, intermediate_size, bias=False, **kwargs)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, bias=False, **kwargs)

    def _weights(self):
        """The projections' weights where calling them is a product with those and nothing else, or None."""
        if calls_are_watched() or _calls() != _CALLS:
            return None
        weights = []
        for name in ('gate_proj', 'up_proj', 'down_proj'):
            m = self._modules[name]
            if not calls_nothing_else(m, nn.Linear):
                return None
            params = m.__dict__['_parameters']
            # (torch.func.functional_call puts plain tensors in the parameters' places)
            if type(params.get('weight')) not in (nn.Parameter, torch.Tensor) or params.get('bias') is not None:
                return None
            weights.append(params['weight'])
        return weights

    def forward(self, x: torch.Tensor, **kwargs) -> torch.Tensor:
        weights = self._weights()
        if weights is not None:
            return gated_mlp(x, *weights, self.hidden_act)
        require_gpu(x)
        gate, up = self.gate_proj(x), self.up_proj(x)
        g = gate.float()
        act = torch.sigmoid(g) if self.hidden_act == 'sigmoid' else F.gelu(g, approximate='tanh') if self.hidden_act == 'gelu_tanh' else F.silu(g)
        return self.down_proj((act * up.float()).to(up.dtype))
