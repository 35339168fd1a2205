"""When the feed-forward block's layer may hand its weights to the operator: only where calling its projections would do nothing else."""
import contextlib

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from fla_hip.modules import mlp as mlp_module
from fla_hip.modules import GatedMLP
from oracle import modules_oracle as M
from oracle.gdn_oracle import get_err_ratio


class Adapter(nn.Module):
    """A projection with a correction of low rank beside it."""

    def __init__(self, base, rank=2):
        super().__init__()
        self.base = base
        self.a, self.b = (nn.Parameter(torch.randn(*s, device=base.weight.device).to(base.weight.dtype) * 0.3) for s in ((rank, base.in_features), (base.out_features, rank)))

    @property
    def weight(self):
        return self.base.weight

    def forward(self, x):
        return self.base(x) + (x @ self.a.t()) @ self.b.t()


class _Dispatch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class _Function(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class _Quantised(nn.Parameter):
    pass


@pytest.fixture
def calls(monkeypatch):
    """The operator's calls (on the CPU: it is the oracle that answers)."""
    made = []

    def operator(x, wg, wu, wd, activation):
        made.append(activation)
        return M.gated_mlp(x, wg, wu, wd, activation, torch.float32)

    monkeypatch.setattr(mlp_module, 'gated_mlp', operator)
    monkeypatch.setattr(mlp_module, 'require_gpu', lambda x, *_: x.device)
    return made


def _layer(act='swish'):
    torch.manual_seed(0)
    return GatedMLP(16, intermediate_size=24, hidden_act=act)


def test_plain_projections_go_to_the_operator(calls):
    layer = _layer()
    x = torch.randn(3, 16)
    y = layer(x)
    with torch.device('cpu'):
        layer(x)
    swapped = torch.func.functional_call(layer, {n: p.detach() * 2 for n, p in layer.named_parameters()}, (x,))
    assert calls == ['swish'] * 3 and not torch.equal(swapped, y)


def _replace(name, make):
    return lambda layer, stack, monkeypatch: setattr(layer, name, make(getattr(layer, name)))


def _biased(m):
    new = nn.Linear(m.in_features, m.out_features, bias=True)
    with torch.no_grad():
        new.weight.copy_(m.weight)
    return new


def _global_hook(register):
    return lambda layer, stack, monkeypatch: stack.callback(register(lambda *a: None).remove)


CHANGES = {
    'adapter of the gate': _replace('gate_proj', Adapter),
    'adapter of up': _replace('up_proj', Adapter),
    'adapter of down': _replace('down_proj', Adapter),
    'bias': _replace('up_proj', _biased),
    'bias of down': _replace('down_proj', _biased),
    'forward': lambda layer, stack, monkeypatch: setattr(layer.gate_proj, 'forward', lambda x, own=layer.gate_proj.forward: own(x)),
    'Linear.forward': lambda layer, stack, monkeypatch: monkeypatch.setattr(nn.Linear, 'forward', lambda self, x: x @ self.weight.t()),
    'F.linear': lambda layer, stack, monkeypatch: monkeypatch.setattr(F, 'linear', lambda x, w, b=None: x @ w.t()),
    'compiled': lambda layer, stack, monkeypatch: setattr(layer.up_proj, '_compiled_call_impl', layer.up_proj._call_impl),
    'forward hook': lambda layer, stack, monkeypatch: layer.down_proj.register_forward_hook(lambda m, a, out: None),
    'forward pre hook': lambda layer, stack, monkeypatch: layer.gate_proj.register_forward_pre_hook(lambda m, a: None),
    'backward hook': lambda layer, stack, monkeypatch: layer.up_proj.register_full_backward_hook(lambda m, a, b: None),
    'global forward hook': _global_hook(nn.modules.module.register_module_forward_hook),
    'parametrised': lambda layer, stack, monkeypatch: torch.nn.utils.parametrize.register_parametrization(layer.up_proj, 'weight', nn.Identity()),
    'other parameter': lambda layer, stack, monkeypatch: setattr(layer.gate_proj, 'weight', _Quantised(layer.gate_proj.weight.detach())),
    'dispatch mode': lambda layer, stack, monkeypatch: stack.enter_context(_Dispatch()),
    'function mode': lambda layer, stack, monkeypatch: stack.enter_context(_Function()),
}


@pytest.mark.parametrize('act', ['swish', 'sigmoid', 'gelu_tanh'])
@pytest.mark.parametrize('change', CHANGES)
def test_projections_that_do_more_are_called(calls, monkeypatch, change, act):
    layer = _layer(act)
    x = torch.randn(5, 16)
    with contextlib.ExitStack() as stack, torch.no_grad():
        CHANGES[change](layer, stack, monkeypatch)
        y = layer(x)
        assert calls == []
        want = layer.down_proj(M.gate_activation(layer.gate_proj(x), act)[0] * layer.up_proj(x))
    torch.testing.assert_close(y, want)


def test_hooks_see_their_calls(calls):
    layer = _layer()
    seen = []
    for name in ('gate_proj', 'up_proj', 'down_proj'):
        getattr(layer, name).register_forward_hook(lambda m, a, out, name=name: seen.append((name, tuple(out.shape))))
    layer(torch.randn(5, 16))
    assert seen == [('gate_proj', (5, 24)), ('up_proj', (5, 24)), ('down_proj', (5, 16))]


def test_cpu_tensors_are_refused_on_either_path():
    layer = _layer()
    layer.gate_proj = Adapter(layer.gate_proj)
    with pytest.raises(RuntimeError, match='GPU'):
        layer(torch.randn(5, 16))


@pytest.mark.gpu
def test_a_block_with_an_adapter_trains():
    """fp32 sums of 256 and 512 terms between roundings to bf16: of g, u (each carried through the activation's slope), h and the result, and of the two parts
    of an adapted projection: 2-norms within 4 u of the same steps in 64 bits for y, and 6 u for the gradients, which meet as many again on the way back."""
    torch.manual_seed(1)
    layer = GatedMLP(256, intermediate_size=512, device='cuda', dtype=torch.bfloat16)
    layer.up_proj = Adapter(layer.up_proj)
    x, dy = (torch.randn(40, 256, device='cuda').bfloat16() for _ in range(2))
    leaves = [x.requires_grad_(True), *layer.parameters()]
    names = ['x', *(n for n, _ in layer.named_parameters())]
    y = layer(x)
    got = torch.autograd.grad(y, leaves, dy)
    t = {n: p.detach().double().requires_grad_(True) for n, p in zip(names, leaves)}
    up = t['x'] @ t['up_proj.base.weight'].t() + (t['x'] @ t['up_proj.a'].t()) @ t['up_proj.b'].t()
    ref = (F.silu(t['x'] @ t['gate_proj.weight'].t()) * up) @ t['down_proj.weight'].t()
    want = torch.autograd.grad(ref, [t[n] for n in names], dy.double())
    u = torch.finfo(torch.bfloat16).eps / 2
    assert get_err_ratio(ref, y.double()) <= 4 * u
    for n, g, w in zip(names, got, want):
        assert get_err_ratio(w, g.double()) <= 6 * u, n
