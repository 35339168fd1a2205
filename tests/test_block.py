"""The block around the Gated DeltaNet layer (fla_hip.layers.GatedDeltaNetBlock): norm, mixing, norm with the residual stream, feed-forward block, run
together as a model does, against the same steps in fp32 torch around the layer itself (which tests/test_layer.py holds against the oracles)."""
import pytest
import torch

from oracle import modules_oracle as M
from oracle.gdn_oracle import get_err_ratio

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF = torch.bfloat16
U = torch.finfo(BF).eps / 2


def _block(seed=0, **kw):
    from fla_hip.layers import GatedDeltaNetBlock
    torch.manual_seed(seed)
    args = dict(hidden_size=256, intermediate_size=500, head_dim=64, num_heads=2, num_v_heads=4, layer_idx=0)
    args.update(kw)
    block = GatedDeltaNetBlock(**args)
    with torch.no_grad():
        for name, p in block.named_parameters():
            if name.endswith('norm.weight'):
                p.normal_(1, 0.2)
    return block.to(DEV).to(BF)


def _r(x):
    """The rounding that a step's result goes through (its gradient passes as it is)."""
    return x + (x.detach().to(BF).float() - x.detach())


def _steps(block, x, **kw):
    """The same block with everything but the mixing layer in fp32 torch, rounded to bf16 where its tensors are."""
    norm = lambda m, r: _r(M.layer_norm(r, m.weight, None, m.eps, True, torch.float32)[0])
    mixed = block.attn(norm(block.attn_norm, x).to(BF), **kw)[0].float()
    stream = _r(x + mixed)
    m = block.mlp
    y = M.gated_mlp(norm(block.mlp_norm, stream), m.gate_proj.weight, m.up_proj.weight, m.down_proj.weight, m.hidden_act, torch.float32)
    return _r(stream + _r(y))


def test_parameter_names_are_the_references():
    names = {n.split('.')[0] for n, _ in _block().named_parameters()}
    assert names == {'attn_norm', 'attn', 'mlp_norm', 'mlp'}
    assert {n for n, _ in _block().mlp.named_parameters()} == {'gate_proj.weight', 'up_proj.weight', 'down_proj.weight'}


@pytest.mark.parametrize(('B', 'T'), [(1, 1), (2, 20), (2, 130), (1, 700)])
def test_forward(B, T):
    block = _block().eval()
    x = torch.randn(B, T, 256, device=DEV).to(BF)
    got = block(x)[0]
    with torch.no_grad():
        want = _steps(block, x.float())
    # the normalisations' roundings may differ by a step here and there (fp32 sums in another order); the layer and the feed-forward block carry that on, and h
    # is rounded on the way: a handful of roundings of u / sqrt(3) each, most of them of the smaller of two summands
    assert get_err_ratio(want, got.float()) <= 2 * U


@pytest.mark.parametrize('T', [65, 300])
def test_backward(T):
    """Gradients of the input and of every parameter against torch's autograd through the same steps.  Between the two runs lie the roundings of the feed-forward
    block's inner gradients (k = 3: u), of the normalisations' (u / sqrt(3) each, three of them) and of dx, all carried through the layer's backward: within
    4 u in the 2-norm."""
    block = _block().train()
    x = torch.randn(2, T, 256, device=DEV).to(BF)
    dy = torch.randn(2, T, 256, device=DEV).to(BF)
    a = x.clone().requires_grad_(True)
    leaves = [a, *block.parameters()]
    got = torch.autograd.grad(block(a)[0], leaves, dy)
    b = x.float().requires_grad_(True)
    leaves = [b, *block.parameters()]
    want = torch.autograd.grad(_steps(block, b), leaves, dy.float())
    for name, g, w in zip(['x', *(n for n, _ in block.named_parameters())], got, want):
        assert get_err_ratio(w.float(), g.float()) <= 4 * U, name


def test_prefill_and_decode_through_the_cache():
    """A prompt, then one token at a time: each step's output against the whole sequence in one go."""
    from fla_hip.layers import LayerCache
    block = _block().eval()
    x = torch.randn(2, 90, 256, device=DEV).to(BF)
    whole = block(x)[0]
    cache = LayerCache()
    out = [block(x[:, :80], past_key_values=cache, use_cache=True)[0]]
    out += [block(x[:, t:t + 1], past_key_values=cache, use_cache=True)[0] for t in range(80, 90)]
    # (the token recurrence instead of the chunked form in the mixing layer: 5e-3, its own bound)
    assert get_err_ratio(whole.float(), torch.cat(out, 1).float()) <= 5e-3
    assert not block(x)[0].requires_grad


def test_a_padded_batch():
    block = _block().eval()
    x = torch.randn(3, 100, 256, device=DEV).to(BF)
    mask = torch.ones(3, 100, dtype=torch.int64, device=DEV)
    mask[0, :40] = 0
    mask[2, :99] = 0
    got = block(x, attention_mask=mask)[0]
    for b, n in ((0, 60), (1, 100), (2, 1)):
        alone = block(x[b:b + 1, 100 - n:])[0]
        assert get_err_ratio(alone.float(), got[b:b + 1, 100 - n:].float()) <= 5e-3, b


@pytest.mark.parametrize('dtype', [BF, torch.float16])
def test_under_autocast(dtype):
    """fp32 weights and an fp32 residual stream, as a training loop under autocast has them: against the same block's weights and input in the 16-bit type.
    The two differ by the roundings of the weights of the norms and of the streams to 16 bits, each u / sqrt(3) in the 2-norm and carried on to the end: the stream
    twice, its sum, the norms' weights twice: within 4 u.  The stream stays in fp32, and every parameter gets a gradient of its own type."""
    block = _block().float().train()
    u = torch.finfo(dtype).eps / 2
    x = torch.randn(2, 130, 256, device=DEV).to(dtype).float().requires_grad_(True)
    with torch.autocast('cuda', dtype=dtype):
        y = block(x)[0]
        assert get_err_ratio(y.detach(), block.eval()(x)[0]) <= 4 * u
    assert y.dtype == torch.float32
    grads = torch.autograd.grad(y, [x, *block.parameters()], torch.randn(y.shape, device=DEV, generator=torch.Generator(DEV).manual_seed(1)))
    assert all(g.dtype == torch.float32 and bool(g.isfinite().all()) and bool(g.any()) for g in grads)
    low = _block().to(dtype).eval()
    assert get_err_ratio(low(x.detach().to(dtype))[0].float(), y.detach()) <= 4 * u
