"""Forward-mode derivatives of the normalisation and of the feed-forward block: there are none, and a dual tensor is refused rather than answered without its
tangent - with a gradient asked for or not, whichever input it is."""
import pytest
import torch
from torch.autograd import forward_ad

from fla_hip import _lib
from fla_hip.modules import layernorm, mlp


class Library:
    def __getattr__(self, name):
        return lambda *a: 4 if name.endswith(('workspace_bytes', 'bwd_parts')) else 0


def _norm(dtype, device):
    t = [torch.randn(*s, device=device).to(dtype) for s in ((5, 64), (64,), (64,), (5, 64))]
    return t, lambda x, w, b, r: layernorm.layer_norm(x, w, b, residual=r)


def _mlp(dtype, device):
    t = [torch.randn(*s, device=device).to(dtype) for s in ((5, 24), (40, 24), (40, 24), (24, 40))]
    return t, mlp.gated_mlp


def _refused(make, which, requires_grad, device):
    t, call = make(torch.bfloat16, device)
    with forward_ad.dual_level():
        call(*t)                                                                # (a level alone changes nothing)
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                args = list(t)
                args[which] = forward_ad.make_dual(t[which].clone().requires_grad_(requires_grad), torch.ones_like(t[which]))
                with pytest.raises(NotImplementedError, match='forward-mode'):
                    call(*args)


@pytest.mark.parametrize('requires_grad', [False, True])
@pytest.mark.parametrize('which', range(4))
@pytest.mark.parametrize('make', [_norm, _mlp])
def test_dual_tensors_are_refused_by_the_python_path(make, which, requires_grad, monkeypatch):
    """(CPU: the library and the device are stand-ins.)"""
    monkeypatch.setattr(_lib, 'load', Library)
    monkeypatch.setattr(_lib, 'host', _lib._PythonHost)
    for m in (layernorm, mlp):
        monkeypatch.setattr(m, 'require_gpu', lambda x, *_: x.device)
        monkeypatch.setattr(m, 'launch', lambda *a: None)
    _refused(make, which, requires_grad, 'cpu')


@pytest.mark.gpu
@pytest.mark.parametrize('requires_grad', [False, True])
@pytest.mark.parametrize('which', range(4))
@pytest.mark.parametrize('make', [_norm, _mlp])
def test_dual_tensors_are_refused(make, which, requires_grad):
    _refused(make, which, requires_grad, 'cuda')
