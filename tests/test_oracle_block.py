"""The oracles of the normalisation and of the feed-forward block: against torch's own functions, and their gradient formulas against
differences (CPU, 64 bits)."""
import pytest
import torch
import torch.nn.functional as F

from oracle import modules_oracle as M

ACTS = ['swish', 'sigmoid', 'gelu_tanh']


def _rand(*shape, seed=0, std=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * std


def _differences(f, t, v, h=1e-5):
    return (f(t + h * v) - f(t - h * v)) / (2 * h)


@pytest.mark.parametrize('D', [1, 2, 17, 96])
def test_norms_are_torchs(D):
    r, w, b = _rand(5, D), _rand(D, seed=1), _rand(D, seed=2)
    torch.testing.assert_close(M.layer_norm(r, w, b, 1e-3)[0], F.layer_norm(r, (D,), w, b, 1e-3))
    torch.testing.assert_close(M.layer_norm(r, w, None, 1e-3, True)[0], F.rms_norm(r, (D,), w, 1e-3))


@pytest.mark.parametrize('rms', [False, True])
@pytest.mark.parametrize('D', [2, 17, 96])
def test_norm_gradients_are_the_differences(D, rms):
    r, w, b, dy, ds = _rand(5, D), _rand(D, seed=1), _rand(D, seed=2), _rand(5, D, seed=3), _rand(5, D, seed=4)
    dr, dw, db = M.layer_norm_grads(r, w, dy, ds, 1e-3, rms)
    y = lambda r, w, b: (M.layer_norm(r, w, b, 1e-3, rms)[0] * dy).sum() + (r * ds).sum()
    for i, (t, g) in enumerate(((r, dr), (w, dw), (b, db))):
        v = _rand(*t.shape, seed=9)
        got = _differences(lambda t: y(*((r, w, b)[:i] + (t,) + (r, w, b)[i + 1:])), t, v)
        # (differences: error h^2 and rounding 1e-16 / h, both near 1e-10 of terms of order 1..D)
        torch.testing.assert_close((g * v).sum(), got, rtol=1e-7, atol=1e-7)


@pytest.mark.parametrize('act', ACTS)
def test_activations_are_torchs(act):
    x = torch.linspace(-30, 30, 2001, dtype=torch.float64)
    a, da = M.gate_activation(x, act)
    want = {'swish': F.silu, 'sigmoid': torch.sigmoid, 'gelu_tanh': lambda x: F.gelu(x, approximate='tanh')}[act]
    torch.testing.assert_close(a, want(x), rtol=1e-9, atol=1e-12)
    leaf = x.clone().requires_grad_(True)
    torch.testing.assert_close(da, torch.autograd.grad(want(leaf).sum(), leaf)[0], rtol=1e-9, atol=1e-12)


@pytest.mark.parametrize('act', ACTS)
def test_mlp_gradients_are_the_differences(act):
    n, D, H = 5, 7, 11
    t = [_rand(n, D), _rand(H, D, seed=1), _rand(H, D, seed=2), _rand(D, H, seed=3)]
    dy = _rand(n, D, seed=4)
    for i, g in enumerate(M.gated_mlp_grads(*t, dy, act)):
        v = _rand(*t[i].shape, seed=9)
        got = _differences(lambda x: (M.gated_mlp(*t[:i], x, *t[i + 1:], act) * dy).sum(), t[i], v)
        torch.testing.assert_close((g * v).sum(), got, rtol=1e-7, atol=1e-7)
