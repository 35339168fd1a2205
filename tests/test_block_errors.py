"""The normalisation's and the feed-forward block's calls that cannot be finished: exceptions that the caller can catch, and the same call succeeds afterwards."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _norm(rows=64, D=256):
    from fla_hip.modules import rms_norm
    x, r, w = (torch.randn(*s, device='cuda').to(BF) for s in ((rows, D), (rows, D), (D,)))
    return x, lambda x: rms_norm(x, w, None, residual=r, prenorm=True)[0]


def _mlp(rows=64, D=256, F=512):
    from fla_hip.modules import gated_mlp
    x, wg, wu, wd = (torch.randn(*s, device='cuda').to(BF) for s in ((rows, D), (F, D), (F, D), (D, F)))
    return x, lambda x: gated_mlp(x, wg, wu, wd)


@pytest.mark.parametrize('make', [_norm, _mlp])
@pytest.mark.parametrize('form', ['vmap', 'func_grad', 'func_jvp', 'sparse', 'fake'])
def test_tensors_without_plain_memory_raise(make, form):
    x, call = make()
    want = call(x)
    with pytest.raises(Exception):
        if form == 'vmap':
            torch.vmap(call)(torch.stack([x, x]))
        elif form == 'func_grad':
            torch.func.grad(lambda x: call(x).float().sum())(x)
        elif form == 'func_jvp':
            torch.func.jvp(call, (x,), (x,))
        elif form == 'sparse':
            call(x.to_sparse())
        else:
            with FakeTensorMode(allow_non_fake_inputs=True) as mode:
                call(mode.from_tensor(x))
    assert torch.equal(call(x), want)


@pytest.mark.parametrize('train', [False, True])
@pytest.mark.parametrize('make', [_norm, _mlp])
def test_out_of_memory_can_be_caught(make, train):
    x, call = make(8192, 2048)
    x.requires_grad_(train)
    want = call(x)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(1e-9)
    try:
        held = []                                       # (blocks that were reserved before still serve small requests)
        with pytest.raises(torch.OutOfMemoryError):
            for _ in range(4096):
                held.append(call(x))
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    held.clear()
    assert torch.equal(call(x), want)


def test_out_of_memory_in_the_backward_can_be_caught():
    x, call = _mlp(8192, 2048, 5632)
    x.requires_grad_(True)
    y = call(x)
    dy = torch.ones_like(y)
    (want,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(1e-9)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            torch.autograd.grad(y, x, dy, retain_graph=True)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
