"""Every call of the normalisation and of the feed-forward block into the library is made with the tensors' device as the current one (CPU: the library and
the device guard are stand-ins that keep record)."""
import contextlib

import pytest
import torch

from fla_hip import _lib
from fla_hip.modules import layernorm, mlp
from fla_hip.ops.gated_delta_rule import _common


class Library:
    def __init__(self):
        self.calls, self.inside = [], 0

    def __getattr__(self, name):
        if name.endswith(('workspace_bytes', 'bwd_parts')):                  # (entries that launch nothing)
            return lambda *a: 4
        return lambda *a: self.calls.append((name, self.inside > 0)) or 0

    @contextlib.contextmanager
    def device(self, dev):
        self.inside += 1
        yield
        self.inside -= 1


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, 'load', lambda: lib)
    monkeypatch.setattr(torch.cuda, 'device', lib.device)
    monkeypatch.setattr(_common, 'current_device', lambda: 7)
    monkeypatch.setattr(_common, 'current_stream_ptr', lambda dev: 0)
    for m in (_common, layernorm, mlp):
        monkeypatch.setattr(m, 'require_gpu', lambda x, *_: x.device)
    return lib


@pytest.mark.parametrize('residual', [False, True])
def test_normalisation(lib, residual):
    x = torch.zeros(5, 64)
    w, b = torch.ones(64), torch.zeros(64)
    _, mean, rstd, r = layernorm.layer_norm_fwd(x, w, b, residual=x if residual else None)
    layernorm.layer_norm_bwd(x, r, w, b, 1e-5, mean, rstd, x, residual)
    assert lib.calls == [(name, True) for name in ('gdn_layer_norm_fwd', 'gdn_layer_norm_bwd', 'gdn_sum_rows')]


@pytest.mark.parametrize('rows', [1, 40])
def test_feed_forward_block(lib, rows):
    x, wg, wu, wd = (torch.zeros(*size, dtype=torch.bfloat16) for size in ((rows, 24), (40, 24), (40, 24), (24, 40)))
    y, s, a, h = mlp._forward(x, wg, wu, wd, _lib.ACT_SILU, True)
    assert y.shape == x.shape and s.shape == a.shape == h.shape == (rows, 40)
    y = mlp.GatedMLPFunction.apply(x.requires_grad_(), wg, wu, wd, _lib.ACT_SILU)
    y.backward(torch.zeros_like(y))
    assert lib.calls == [(name, True) for name in ('gdn_gated_mlp_fwd', 'gdn_gated_mlp_fwd', 'gdn_gated_mlp_bwd')]
