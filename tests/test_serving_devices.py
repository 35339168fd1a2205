"""Every call of a serving step's operators into the library is made with the tensors' device as the current one, and with the sizes that it says (CPU: the library and
the device guard are stand-ins that keep record)."""
import contextlib

import pytest
import torch

from fla_hip import _lib
from fla_hip.modules import rotary
from fla_hip.ops.attn import paged
from fla_hip.ops.drafts import verify
from fla_hip.ops.gated_delta_rule import _common

BF = torch.bfloat16


class Library:
    def __init__(self):
        self.calls, self.inside = [], 0

    def __getattr__(self, name):
        if name.endswith('workspace_bytes'):                  # (entries that launch nothing)
            return lambda *a: 64
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
    monkeypatch.setattr(_lib, 'host', lambda: _lib._PythonHost)
    monkeypatch.setattr(torch.cuda, 'device', lib.device)
    monkeypatch.setattr(_common, 'current_device', lambda: 7)
    monkeypatch.setattr(_common, 'current_stream_ptr', lambda dev: 0)
    for m in (rotary, paged, verify):
        monkeypatch.setattr(m, 'require_gpu', lambda x, *_: x.device)
    return lib


def test_rotary(lib):
    x, cos = torch.zeros(2, 4, 3, 16, dtype=BF, requires_grad=True), torch.zeros(8, 8)
    y = rotary.rotary_embedding(x, cos, cos)
    y.backward(torch.zeros_like(y))
    rotary.RotaryEmbedding(16, scale_base=512.0)(x.detach(), x.detach())
    assert lib.calls == [('gdn_rotary', True)] * 4


def test_step(lib):
    kc, vc = torch.zeros(2, 5, 8, 2, 64, dtype=BF)
    table, context = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q, k, cos = torch.zeros(2, 4, 4, 64, dtype=BF), torch.zeros(2, 4, 2, 64, dtype=BF), torch.zeros(30, 32)
    at = kc._version
    assert paged.paged_append(k, k, kc, vc, table, context, q=q, cos=cos, sin=cos).shape == q.shape
    assert kc._version > at
    assert paged.paged_attn(q, kc, vc, table, context).shape == q.shape
    at = vc._version
    paged.paged_keep(kc, vc, table, context, torch.zeros(2, 4, dtype=torch.int32), context)
    assert vc._version > at
    p = torch.zeros(2, 4, 9)
    token, kept, rows = verify.verify_drafts(p, torch.zeros(2, 4, dtype=torch.int64), torch.zeros(2, 4))
    assert (token.shape, kept.shape, rows.shape) == ((2,), (2,), (2, 4)) and (token.dtype, kept.dtype, rows.dtype) == (torch.int64, torch.int32, torch.int32)
    assert lib.calls == [(name, True) for name in ('gdn_paged_append', 'gdn_paged_attn', 'gdn_paged_keep', 'gdn_verify_drafts')]
