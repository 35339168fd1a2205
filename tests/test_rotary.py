"""Rotary positions (fla_hip.modules: rotary_embedding, rotary_embedding_qk, RotaryEmbedding) against the 64-bit oracle, element by element.

Tolerance, u = half the spacing of the result's type relative to it, e = 2^-24: two products and a sum in fp32, three roundings of at most e of the magnitudes
that enter (|x1 c| + |x2 s|), and one rounding of the result, u |ref|; results below the smallest normal number of fp16 are off by half its smallest step, 2^-25."""
import math

import pytest
import torch

from oracle import serving_oracle as O

gpu = pytest.mark.gpu
DEV = 'cuda'
E = 2.0 ** -24
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _mods():
    import fla_hip.modules as mods
    return mods


def _near(name, got, ref, size):
    assert tuple(got.shape) == tuple(ref.shape), (name, got.shape, ref.shape)
    got = got.detach().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), name
    ok = ~ref.isnan()
    u = torch.finfo(got.dtype).eps / 2
    tol = u * ref.abs() * (1 + 1e-3) + 3 * E * size + (2.0 ** -25 if got.dtype == HF else 2.0 ** -140)
    worst = ((got.double() - ref).abs()[ok] / tol[ok]).max().item() if ok.any() else 0.0
    assert worst <= 1, f'{name}: {worst:.2f} of the tolerance'


def _tables(positions, R, dtype=FP, seed=0):
    t = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return t.cos().to(dtype).to(DEV), t.sin().to(dtype).to(DEV)


def _rows(*shape, dtype, seed=0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * 2).to(dtype).to(DEV)


# head sizes and turned parts on every side of a thread's 16 bytes
HEADS = [(2, 2), (8, 8), (64, 64), (64, 32), (80, 80), (72, 72), (128, 128), (128, 2), (128, 50), (100, 100), (256, 256), (256, 64), (96, 90), (34, 18), (1024, 1024)]


@gpu
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dtype', [BF, HF, FP])
@pytest.mark.parametrize(('D', 'R'), HEADS)
def test_against_the_oracle(D, R, dtype, interleaved):
    B, T, HQ, HK = 2, 5, 3, 1
    cos, sin = _tables(T + 3, R)
    q, k = _rows(B, T, HQ, D, dtype=dtype, seed=D), _rows(B, T, HK, D, dtype=dtype, seed=R)
    at = torch.arange(T).expand(B, T) + 3
    got = _mods().rotary_embedding_qk(q, k, cos, sin, interleaved=interleaved, seqlen_offsets=3)
    for name, x, y in (('q', q, got[0]), ('k', k, got[1])):
        assert y.dtype == dtype
        _near(name, y, *O.rotary(x, cos, sin, at, interleaved))


@gpu
@pytest.mark.parametrize(('T', 'HQ', 'HK', 'D'), [(1, 1, 1, 64), (1, 32, 8, 128), (777, 5, 1, 64), (300, 20, 4, 128), (130, 71, 1, 40), (3000, 8, 8, 128), (9, 300, 7, 256)])
def test_sizes_from_a_row_to_a_full_chip(T, HQ, HK, D):
    cos, sin = _tables(T, D)
    q, k = _rows(1, T, HQ, D, dtype=BF), _rows(1, T, HK, D, dtype=BF, seed=1)
    got = _mods().rotary_embedding_qk(q, k, cos, sin)
    for x, y in zip((q, k), got):
        a, b = x.double()[..., :D // 2], x.double()[..., D // 2:]
        c, s = cos.double()[:, None], sin.double()[:, None]
        _near('x', y, torch.cat([a * c - b * s, a * s + b * c], -1).cpu(), torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1).cpu())


@gpu
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
@pytest.mark.parametrize('cu', [[0, 7], [0, 0, 3, 3, 4, 7], [1, 2, 5], [0, 1, 2, 3, 4, 5, 6, 7]])
def test_packed_batches(cu, index):
    T = 7
    cos, sin = _tables(40, 64)
    x = _rows(1, T, 2, 64, dtype=BF)
    bounds = torch.tensor(cu, dtype=index, device=DEV)
    N = len(cu) - 1
    offsets = torch.arange(N) * 5
    at = torch.full((1, T), -1)
    for n in range(N):
        at[0, cu[n]:cu[n + 1]] = torch.arange(cu[n + 1] - cu[n]) + offsets[n]
    for max_seqlen in (None, T):
        y = _mods().rotary_embedding(x, cos, sin, cu_seqlens=bounds, seqlen_offsets=offsets.to(DEV).to(index), max_seqlen=max_seqlen)
        _near('packed', y, *O.rotary(x, cos, sin, at))


@gpu
@pytest.mark.parametrize('heads', [2, 20])
@pytest.mark.parametrize('N', [1, 63, 64, 130, 700])
def test_many_sequences(N, heads):
    """Some of them empty, rows before the first and behind the last; tokens of few threads and of many."""
    lengths = torch.randint(0, 4, (N,), generator=torch.Generator().manual_seed(N))
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]) + 3
    T = int(cu[-1]) + 2
    at = torch.full((1, T), -1)
    for n in range(N):
        at[0, cu[n]:cu[n + 1]] = torch.arange(lengths[n]) + n % 30
    cos, sin = _tables(40, 128)
    x = _rows(1, T, heads, 128, dtype=BF)
    y = _mods().rotary_embedding(x, cos, sin, cu_seqlens=cu.to(DEV), seqlen_offsets=(torch.arange(N) % 30).to(DEV), max_seqlen=T)
    _near('many', y, *O.rotary(x, cos, sin, at))


@gpu
@pytest.mark.parametrize('index', [torch.int32, torch.int64, torch.int16])
def test_positions_and_those_the_tables_do_not_have(index):
    cos, sin = _tables(10, 32)
    x = _rows(2, 4, 2, 40, dtype=HF)
    positions = torch.tensor([[9, 0, 3, 3], [10, 1, 2000, 9]], dtype=index, device=DEV)
    y = _mods().rotary_embedding(x, cos, sin, positions=positions)
    _near('positions', y, *O.rotary(x, cos, sin, positions.cpu()))
    assert y.isnan().any(-1).sum() == 4
    y = _mods().rotary_embedding(x, cos, sin, seqlen_offsets=torch.tensor([-1, 6], dtype=torch.int32, device=DEV))
    assert y[0, 0, :, :32].isnan().all() and torch.equal(y[0, 0, :, 32:], x[0, 0, :, 32:])
    _near('offsets', y[:, 1:], *O.rotary(x[:, 1:], cos, sin, torch.tensor([[0, 1, 2], [7, 8, 9]])))


@gpu
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dtype', [BF, HF])
def test_tables_of_the_rows_type(dtype, interleaved):
    cos, sin = _tables(6, 64, dtype)
    x = _rows(1, 6, 3, 64, dtype=dtype)
    _near('x', _mods().rotary_embedding(x, cos, sin, interleaved=interleaved), *O.rotary(x, cos, sin, torch.arange(6)[None], interleaved))


def _strided(x, how):
    """The numbers of x at other places."""
    B, T, H, D = x.shape
    if how == 'heads_first':
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if how == 'between_16_bytes':
        return torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape)
    if how == 'part_of_a_row':                                   # the middle of a wider projection
        wide = torch.zeros(B, T, 3 * H * D + 5, dtype=x.dtype, device=x.device)
        wide[..., H * D:2 * H * D] = x.flatten(2)
        return wide[..., H * D:2 * H * D].view(B, T, H, D)
    return x.transpose(2, 3).contiguous().transpose(2, 3)        # a head's elements apart


@gpu
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('how', ['heads_first', 'between_16_bytes', 'part_of_a_row', 'elements_apart'])
def test_strides_and_alignments(how, interleaved):
    cos, sin = _tables(9, 64)
    x = _rows(2, 9, 4, 64, dtype=BF)
    want = _mods().rotary_embedding(x, cos, sin, interleaved=interleaved)
    view = _strided(x, how)
    assert torch.equal(view, x)
    assert torch.equal(_mods().rotary_embedding(view, cos, sin, interleaved=interleaved), want)
    wide = torch.zeros(9, 200, device=DEV)                       # tables as parts of a wider tensor, at any address
    wide[:, 3:35], wide[:, 40:72] = cos, sin
    assert torch.equal(_mods().rotary_embedding(x, wide[:, 3:35], wide[:, 40:72], interleaved=interleaved), want)
    if how != 'elements_apart':
        assert _mods().rotary_embedding(view, cos, sin, interleaved=interleaved, inplace=True) is view
        assert torch.equal(view, want)


@gpu
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize(('dtype', 'D', 'R'), [(BF, 128, 128), (HF, 64, 32), (FP, 36, 34)])
def test_gradients_of_a_packed_batch(dtype, D, R, interleaved):
    T, cu = 11, [0, 4, 4, 9]
    cos, sin = _tables(30, R)
    q, k = (_rows(1, T, h, D, dtype=dtype, seed=h).requires_grad_() for h in (3, 1))
    offsets = torch.tensor([0, 7, 20], device=DEV)
    at = torch.tensor([[0, 1, 2, 3, 20, 21, 22, 23, 24, -1, -1]])
    out = _mods().rotary_embedding_qk(q, k, cos, sin, interleaved=interleaved, seqlen_offsets=offsets, cu_seqlens=torch.tensor(cu, device=DEV))
    douts = [_rows(1, T, h, D, dtype=dtype, seed=10 + h) for h in (3, 1)]
    grads = torch.autograd.grad(out, [q, k], douts)
    for x, y, dy, dx in zip((q, k), out, douts, grads):
        _near('y', y, *O.rotary(x.detach(), cos, sin, at, interleaved))
        assert dx.dtype == dtype
        _near('dx', dx, *O.rotary(dy, cos, sin, at, interleaved, back=True))


@gpu
def test_gradients_against_differences_and_of_gradients():
    cos, sin = _tables(5, 8)
    x = _rows(1, 5, 2, 10, dtype=FP).requires_grad_()
    op = lambda x: _mods().rotary_embedding(x, cos, sin)
    dy = _rows(1, 5, 2, 10, dtype=FP, seed=1)
    (dx,) = torch.autograd.grad(op(x), x, dy)
    for i in range(0, x.numel(), 7):
        step = torch.zeros(x.numel(), device=DEV)
        step[i] = 0.5                                            # (linear: any step; the difference of sums of 100 products in fp32)
        there, back = ((op(x.detach() + s * step.view_as(x)).double() * dy.double()).sum() for s in (1, -1))
        assert abs((there - back) - dx.flatten()[i].double()) < 1e-4
    # a gradient of the gradient: the turn itself
    v = _rows(1, 5, 2, 10, dtype=FP, seed=2).requires_grad_()
    (dx,) = torch.autograd.grad(op(x), x, v, create_graph=True)
    (dv,) = torch.autograd.grad(dx, v, dy)
    assert torch.equal(dv, op(dy))


@gpu
def test_broadcast_and_absent_gradients():
    cos, sin = _tables(4, 16)
    q, k = (_rows(2, 4, 2, 16, dtype=BF, seed=s).requires_grad_() for s in (0, 1))
    a, b = _mods().rotary_embedding_qk(q, k, cos, sin)
    dq, dk = torch.autograd.grad(a.float().sum(), [q, k], allow_unused=True)     # (a gradient of ones without memory of its own; none for k)
    assert dk is None
    _near('dq', dq, *O.rotary(torch.ones_like(q), cos, sin, torch.arange(4).expand(2, 4), back=True))
    shared = _rows(2, 4, 1, 16, dtype=BF).requires_grad_()
    y = _mods().rotary_embedding(shared.expand(2, 4, 3, 16), cos, sin)
    (dx,) = torch.autograd.grad(y, shared, torch.ones_like(y))
    one, size = O.rotary(torch.ones(2, 4, 1, 16), cos, sin, torch.arange(4).expand(2, 4), back=True)
    # (three equal gradients in bf16, added up by torch in bf16: two roundings more)
    assert ((dx.double().cpu() - 3 * one).abs() <= 3 * 2.0 ** -8 * (3 * one).abs() + 9 * E * size).all()


@gpu
def test_in_place_under_autograd():
    cos, sin = _tables(4, 16)
    x = _rows(1, 4, 2, 16, dtype=FP)
    leaf = x.clone().requires_grad_()
    y = leaf * 1
    z = _mods().rotary_embedding(y, cos, sin, inplace=True)
    assert z.data_ptr() == y.data_ptr() and torch.equal(z, _mods().rotary_embedding(x, cos, sin))
    (dx,) = torch.autograd.grad(z, leaf, x)
    assert torch.equal(dx, torch.autograd.grad(_mods().rotary_embedding(leaf, cos, sin), leaf, x)[0])
    with pytest.raises(RuntimeError):
        _mods().rotary_embedding(leaf, cos, sin, inplace=True)
    # what a graph has saved and is then turned in place cannot be used by its backward
    saved = x.clone()
    loss = (leaf * saved).sum()
    _mods().rotary_embedding(saved, cos, sin, inplace=True)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


@gpu
def test_replayed_graph_of_a_training_step():
    cos, sin = _tables(64, 64)
    q, k, dq, dk = (_rows(2, 64, h, 64, dtype=BF, seed=i) for i, h in enumerate((4, 2, 4, 2)))
    q.requires_grad_(), k.requires_grad_()

    def step():
        out = _mods().rotary_embedding_qk(q, k, cos, sin, interleaved=True)
        return [*(y.detach() for y in out), *torch.autograd.grad(out, [q, k], [dq, dk])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        with torch.no_grad():
            for t in (q, k, dq, dk):
                t.copy_(_rows(*t.shape, dtype=BF, seed=20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


@gpu
@pytest.mark.parametrize('interleaved', [False, True])
def test_module(interleaved):
    mods = _mods()
    rope = mods.RotaryEmbedding(64, interleaved=interleaved)
    q, k = _rows(2, 20, 4, 96, dtype=BF), _rows(2, 20, 2, 96, dtype=BF, seed=1)
    angle = lambda n: torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    for offset in (0, 100000):
        a, b = rope(q, k, seqlen_offset=offset)
        t = angle(offset + 20)
        at = torch.arange(20).expand(2, 20) + offset
        cos, sin = t.cos().float(), t.sin().float()
        _near('q', a, *O.rotary(q, cos, sin, at, interleaved))
        _near('k', b, *O.rotary(k, cos, sin, at, interleaved))
    one = rope(q[:, :1], k[:, :1], seqlen_offset=torch.tensor([5, 9], device=DEV), max_seqlen=10)
    _near('step', one[0], *O.rotary(q[:, :1], cos, sin, torch.tensor([[5], [9]]), interleaved))
    assert not rope.state_dict() and rope._tables[0].shape[0] == 100020
    with pytest.raises(ValueError, match='max_seqlen'):
        rope(q, k, seqlen_offset=torch.tensor([5, 9], device=DEV))
    # the keys' scale is the inverse of the queries'
    x = mods.RotaryEmbedding(64, scale_base=512.0, interleaved=interleaved)
    a, b = x(q.float(), k.float())
    s = ((torch.arange(0, 64, 2, dtype=torch.float64) + 0.4 * 64) / (1.4 * 64)) ** ((torch.arange(20, dtype=torch.float64) - 10) / 512)[:, None]
    t = angle(20)
    at = torch.arange(20).expand(2, 20)
    _near('q', a, *O.rotary(q.float(), (t.cos() * s).float(), (t.sin() * s).float(), at, interleaved))
    _near('k', b, *O.rotary(k.float(), (t.cos() / s).float(), (t.sin() / s).float(), at, interleaved))


@gpu
def test_module_under_capture_wants_its_tables_first():
    rope = _mods().RotaryEmbedding(64)
    q, k = _rows(1, 8, 2, 64, dtype=BF), _rows(1, 8, 1, 64, dtype=BF)
    rope(q, k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match='before the capture'):
            rope(q, k, seqlen_offset=100)
        held = rope(q, k)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, rope(q, k)))


@gpu
@pytest.mark.parametrize('scale_base', [None, 512.0])
def test_module_keeps_the_tables_of_captured_graphs(scale_base):
    rope = _mods().RotaryEmbedding(64, scale_base=scale_base)
    q, k = _rows(1, 8, 2, 64, dtype=BF), _rows(1, 8, 1, 64, dtype=BF)
    want = rope(q, k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rope(q, k)
    for positions in (300, 50, 4000):
        rope(*(x.repeat(1, positions, 1, 1) for x in (q, k)))
        taken = [torch.full((n, 32), 7.0, device=DEV) for n in (8, 8, 8, 8, 300 * 8, 300 * 8)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), positions
        del taken


@gpu
def test_empty_calls():
    mods = _mods()
    cos, sin = torch.ones(4, 8, device=DEV), torch.zeros(4, 8, device=DEV)
    for shape in ((0, 3, 2, 16), (2, 0, 2, 16), (2, 3, 0, 16)):
        x = torch.zeros(*shape, dtype=BF, device=DEV, requires_grad=True)
        y, z = mods.rotary_embedding_qk(x, x.detach(), cos, sin)
        assert y.shape == z.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape
    # no keys beside the queries
    q = _rows(2, 3, 2, 16, dtype=BF)
    y, z = mods.rotary_embedding_qk(q, q[:, :, :0], cos, sin)
    assert torch.equal(y, q) and z.shape == (2, 3, 0, 16)


@pytest.mark.parametrize('kind', ['linear', 'ntk', 'yarn'])
def test_frequencies_of_stretched_contexts(kind):
    """What each of them is for: the slowest pair turns `factor` times as slowly, and, but for the first, the fastest as fast as before."""
    from fla_hip.modules.rotary import rotary_frequencies
    plain, one = rotary_frequencies(128)
    inv, m = rotary_frequencies(128, scaling=dict(type=kind, factor=4.0, original_max_position_embeddings=8192))
    assert one == 1.0 and inv.dtype == torch.float64 and torch.equal(plain, 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128))
    assert inv[-1].item() == pytest.approx(plain[-1].item() / 4, rel=1e-12)
    assert inv[0].item() == pytest.approx(plain[0].item() / (4 if kind == 'linear' else 1), rel=1e-12)
    assert (inv <= plain).all() and (inv >= plain / 4 * (1 - 1e-12)).all()
    assert m == (pytest.approx(0.1 * math.log(4) + 1) if kind == 'yarn' else 1.0)
    if kind == 'yarn':
        turns = 8192 * plain / (2 * math.pi)
        assert torch.equal(inv[turns > 33], plain[turns > 33]) and torch.allclose(inv[turns < 0.8], plain[turns < 0.8] / 4, rtol=1e-12)


@pytest.mark.parametrize('scaling', [dict(type='linear', factor=0.5), dict(type='other', factor=2.0), dict(type='linear', factor=math.nan)])
def test_frequencies_refuse(scaling):
    from fla_hip.modules.rotary import rotary_frequencies
    with pytest.raises(ValueError):
        rotary_frequencies(64, scaling=scaling)
    with pytest.raises(ValueError):
        rotary_frequencies(63)


class _Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append(name) or 0


@pytest.fixture
def lib(monkeypatch):
    """The library is a stand-in that keeps record: nothing may be launched for a call that is refused."""
    from fla_hip import _lib
    from fla_hip.modules import rotary
    from fla_hip.ops.gated_delta_rule import _common
    lib = _Library()
    monkeypatch.setattr(_lib, 'load', lambda: lib)
    monkeypatch.setattr(_lib, 'host', lambda: _lib._PythonHost)
    monkeypatch.setattr(_common, 'current_device', lambda: None)
    monkeypatch.setattr(_common, 'current_stream_ptr', lambda dev: 0)
    monkeypatch.setattr(rotary, 'require_gpu', lambda x, *_: x.device)
    return lib


def test_refusals(lib):
    op = _mods().rotary_embedding
    x, cos = torch.zeros(2, 4, 3, 16, dtype=BF), torch.zeros(8, 8)
    assert op(x, cos, cos).shape == x.shape and lib.calls == ['gdn_rotary']
    bad = [
        (ValueError, lambda: op(x[0], cos, cos)), (ValueError, lambda: op(x, cos[0], cos[0])), (ValueError, lambda: op(x, cos, cos[:4])),
        (ValueError, lambda: op(x, torch.zeros(8, 9), torch.zeros(8, 9))), (ValueError, lambda: op(x, torch.zeros(8, 0), torch.zeros(8, 0))),
        (ValueError, lambda: op(x, cos[:3], cos[:3])), (ValueError, lambda: op(x, cos, cos, seqlen_offsets=5)), (ValueError, lambda: op(x, cos, cos, seqlen_offsets=-1)),
        (ValueError, lambda: op(x, cos, cos, seqlen_offsets=torch.zeros(3, dtype=torch.int32))), (ValueError, lambda: op(x, cos, cos, seqlen_offsets=torch.zeros(2))),
        (ValueError, lambda: op(x, cos, cos, positions=torch.zeros(4, dtype=torch.int32))), (ValueError, lambda: op(x, cos, cos, positions=torch.zeros(2, 4, dtype=torch.int32), seqlen_offsets=1)),
        (ValueError, lambda: op(x, cos, cos, cu_seqlens=torch.tensor([0, 4]))), (ValueError, lambda: op(x[:1], cos, cos, cu_seqlens=torch.tensor([0, 5]))),
        (ValueError, lambda: op(x[:1], cos, cos, cu_seqlens=torch.tensor([0]))), (ValueError, lambda: op(x[:1], cos, cos, cu_seqlens=torch.tensor([0, 3, 2]))),
        (ValueError, lambda: op(x.transpose(2, 3).contiguous().transpose(2, 3), cos, cos, inplace=True)), (ValueError, lambda: op(x[:, :, :1].expand(2, 4, 3, 16), cos, cos, inplace=True)),
        (NotImplementedError, lambda: op(x.double(), cos, cos)), (NotImplementedError, lambda: op(x, cos.clone().requires_grad_(), cos)),
        (ValueError, lambda: _mods().rotary_embedding_qk(x, x[:1], cos, cos)), (ValueError, lambda: _mods().rotary_embedding_qk(x, x.float(), cos, cos)),
        (ValueError, lambda: _mods().rotary_embedding_qk(x, x[..., :8], cos, cos)),
        (ValueError, lambda: _mods().rotary_embedding_qk(x, x, cos, cos, inplace=True)),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    assert lib.calls == ['gdn_rotary']
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            op(torch.autograd.forward_ad.make_dual(x, x), cos, cos)
    with pytest.raises(NotImplementedError):
        _mods().RotaryEmbedding(16, pos_idx_in_fp32=False)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match='ROCm GPU'):
        _mods().rotary_embedding(torch.zeros(1, 1, 1, 8), torch.zeros(1, 4), torch.zeros(1, 4))


def test_library_refuses():
    """Sizes that no kernel is made for, at the C entry: an error before any launch."""
    import ctypes
    from fla_hip import _lib
    lib = _lib.load()
    rows = _lib.RotaryRows(1, 1, 1)

    def call(**kw):
        c = _lib.RotaryCall(cos=16, sin=16, table_rows=4, table_stride=8, B=1, T=1, N=1, D=16, rotary_dim=16, dtype=0, table_dtype=2)
        for k, v in kw.items():
            setattr(c, k, v)
        return lib.gdn_rotary(ctypes.byref(rows), 1, ctypes.byref(c), None)

    invalid = [dict(B=-1), dict(T=-1), dict(D=0), dict(rotary_dim=15), dict(rotary_dim=18), dict(table_stride=7), dict(cos=None), dict(cu_seqlens=16, B=2), dict(cu_seqlens=16, N=0), dict(table_dtype=1)]
    assert [call(**kw) for kw in invalid] == [_lib.GDN_ERR_INVALID] * len(invalid)
    unsupported = [dict(D=1026), dict(dtype=3), dict(D=17, flags=_lib.ROTARY_INTERLEAVED), dict(B=2 ** 31), dict(T=2 ** 31), dict(B=2 ** 16, T=2 ** 16), dict(T=2 ** 28, D=1024)]
    assert [call(**kw) for kw in unsupported] == [_lib.GDN_ERR_UNSUPPORTED] * len(unsupported)
    assert lib.gdn_rotary(ctypes.byref(rows), 3, ctypes.byref(_lib.RotaryCall(B=1, T=1, D=16)), None) == _lib.GDN_ERR_INVALID
    assert lib.gdn_rotary(ctypes.byref(rows), 1, None, None) == _lib.GDN_ERR_INVALID
    assert call(B=0) == call(T=0) == _lib.GDN_OK


# what a saved-tensor hook may hand back: another type, another place, another layout
HOOKS = {'types': lambda x: x.double() if x.is_floating_point() else x.to(torch.int64 if x.dtype == torch.int32 else torch.int16), 'layout': lambda x: torch.stack([x, x], -1)[..., 0], 'host': lambda x: x.cpu()}


def _seen(c):
    """What a kernel reads behind the pointers of a call (CPU tensors): tables, positions, offsets, boundaries."""
    import ctypes
    read = lambda at, n, of: list((of * n).from_address(at)) if at else None
    index = lambda at, n, is_i32: read(at, n, ctypes.c_int32 if is_i32 else ctypes.c_int64)
    tables = [[read(t + 4 * r * c.table_stride, c.rotary_dim // 2, ctypes.c_float) for r in range(c.table_rows)] for t in (c.cos, c.sin)]
    flags = c.flags
    return (c.table_dtype, c.table_rows, c.rotary_dim, *tables, index(c.positions, c.B * c.T, flags >> 26 & 1), index(c.offsets, c.N, flags >> 27 & 1), index(c.cu_seqlens, c.N + 1, flags >> 5 & 1))


@pytest.mark.parametrize('hook', ['types', 'layout'])
@pytest.mark.parametrize('how', ['positions', 'packed'])
def test_saved_tensors_of_other_types_and_layouts_on_the_host(lib, how, hook):
    """The tables and indices that the gradient's call reads are those of the call itself."""
    calls = []
    lib.gdn_rotary = lambda rows, count, call, stream: calls.append(_seen(call._obj)) or 0
    x = torch.zeros(1, 6, 2, 16, dtype=BF, requires_grad=True)
    wide = torch.rand(10, 40)
    cos, sin = wide[:, 1:9], wide[:, 20:28]
    kw = dict(positions=torch.tensor([[3, 0, 9, 1, 1, 2]], dtype=torch.int32)) if how == 'positions' else dict(cu_seqlens=torch.tensor([0, 2, 6]), seqlen_offsets=torch.tensor([1, 3], dtype=torch.int32))
    for unpack, error in ((lambda t: t, None), (HOOKS[hook], None), (lambda t: t[:-1] if t.dim() == 1 else t[:, :-1], ValueError)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = _mods().rotary_embedding(x, cos, sin, **kw)
        if error is None:
            torch.autograd.grad(y, x, torch.zeros_like(y))
            assert calls[0] == calls[1] and len(calls) == 2
        else:
            with pytest.raises(error, match='came back'):
                torch.autograd.grad(y, x, torch.zeros_like(y))
            assert len(calls) == 1
        calls.clear()


@gpu
@pytest.mark.parametrize('native', [True, False])
@pytest.mark.parametrize('hook', list(HOOKS))
def test_saved_tensors_of_other_types_places_and_layouts(hook, native, monkeypatch):
    from fla_hip import _lib
    if not native:
        monkeypatch.setattr(_lib, 'host', lambda: _lib._PythonHost)
    cos, sin = _tables(30, 64)
    q, k = (_rows(1, 11, h, 64, dtype=BF, seed=h).requires_grad_() for h in (3, 1))
    dy = [_rows(1, 11, h, 64, dtype=BF, seed=10 + h) for h in (3, 1)]
    for kw in (dict(positions=torch.arange(11, dtype=torch.int32, device=DEV)[None] * 2), dict(seqlen_offsets=torch.tensor([0, 7], device=DEV), cu_seqlens=torch.tensor([0, 4, 11], dtype=torch.int32, device=DEV), max_seqlen=7)):
        want = torch.autograd.grad(_mods().rotary_embedding_qk(q, k, cos, sin, **kw), [q, k], dy)
        with torch.autograd.graph.saved_tensors_hooks(HOOKS[hook], lambda t: t):
            out = _mods().rotary_embedding_qk(q, k, cos, sin, **kw)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, [q, k], dy), want))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:-1] if t.dim() == 1 else t[:, :-1]):
            out = _mods().rotary_embedding_qk(q, k, cos, sin, **kw)
        with pytest.raises(ValueError, match='came back'):
            torch.autograd.grad(out, [q, k], dy)


def test_scales_of_calls_that_go_on_from_others(lib):
    """The scale of a query and that of a key it meets cancel only around the same centre: around the middle of each call, other calls' keys raise; around a given one all
    tables begin alike."""
    x = torch.zeros(1, 2, 1, 64, dtype=BF)
    rope = _mods().RotaryEmbedding(64, scale_base=512.0)
    assert rope(x, x)[0].shape == x.shape and len(lib.calls) == 2
    for kw in (dict(seqlen_offset=1), dict(seqlen_offset=torch.zeros(1, dtype=torch.int32), max_seqlen=9), dict(positions=torch.zeros(1, 2, dtype=torch.int32), max_seqlen=9)):
        with pytest.raises(ValueError, match='scale_center'):
            rope(x, x, **kw)
    assert len(lib.calls) == 2
    with pytest.raises(ValueError, match='scale_base'):
        _mods().RotaryEmbedding(64, scale_center=0)
    rope = _mods().RotaryEmbedding(64, scale_base=512.0, scale_center=100)
    tables = {n: rope.tables(n, 'cpu') for n in (1, 40, 300)}
    again = _mods().RotaryEmbedding(64, scale_base=512.0, scale_center=100).tables(300, 'cpu')
    for n, t in tables.items():
        assert all(a.shape[0] >= n and torch.equal(a[:n], b[:n]) for a, b in zip(t, again))
    assert rope.tables(250, 'cpu')[0] is rope.tables(300, 'cpu')[0]
    s = ((torch.arange(0, 64, 2, dtype=torch.float64) + 0.4 * 64) / (1.4 * 64)) ** ((torch.arange(300, dtype=torch.float64) - 100) / 512)[:, None]
    assert torch.equal(again[0], ((torch.arange(300, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).cos() * s).float())


@gpu
def test_token_by_token_around_one_centre():
    """Rows of one whole call, and the same token by token: bit for bit, so every score is the same."""
    q, k = _rows(2, 40, 4, 64, dtype=BF), _rows(2, 40, 2, 64, dtype=BF, seed=1)
    whole = _mods().RotaryEmbedding(64, scale_base=512.0, scale_center=20)
    want = whole(q, k)
    middle = _mods().RotaryEmbedding(64, scale_base=512.0)(q, k)
    assert all(torch.equal(a, b) for a, b in zip(want, middle))
    rope = _mods().RotaryEmbedding(64, scale_base=512.0, scale_center=20)
    for t in range(40):
        offset = t if t % 2 else torch.tensor([t, t], device=DEV)
        got = rope(q[:, t:t + 1], k[:, t:t + 1], seqlen_offset=offset, max_seqlen=1 if t % 2 else 40)
        assert all(torch.equal(a, b[:, t:t + 1]) for a, b in zip(got, want)), t


@pytest.mark.parametrize('center', [None, 0, 3000])
def test_scales_beyond_the_range_of_their_tables(center):
    """(2/7) ** (126 scale_base / log2(7/2)) is 2^-126, the smallest normal number of fp32: at scale_base 64 reached 4461.8 positions from the centre."""
    rope = _mods().RotaryEmbedding(64, scale_base=64.0, scale_center=center)
    most = {None: 8923, 0: 4462, 3000: 7462}[center]
    for n in (most // 2 + 1, most):                              # (the second of them would double the first's)
        assert all(t.isfinite().all() and (torch.maximum(t[:, 0].abs(), t[:, 32].abs()) > 0).all() for t in (torch.cat(pair, 1) for pair in zip(*[iter(rope.tables(n, 'cpu'))] * 2)))
    assert rope.tables(most, 'cpu')[0].shape[0] == most
    with pytest.raises(ValueError, match='range of fp32'):
        rope.tables(most + 2, 'cpu')
    with pytest.raises(ValueError, match='range of fp32'):
        _mods().RotaryEmbedding(64, scale_base=64.0, scale_center=4462).tables(1, 'cpu')


@pytest.mark.parametrize('scaling', [dict(type='yarn', factor=4.0, original_max_position_embeddings=4096, mscale=1.0), dict(type='yarn', factor=4.0, original_max_position_embeddings=4096, mscale_all_dim=0.7),
                                     dict(type='yarn', factor=4.0, original_max_position_embeddings=4096, truncate=False), dict(type='linear', factor=4.0, beta_fast=16), dict(type='ntk', factor=4.0, attention_factor=1.2),
                                     dict(rope_type='linear', factor=4.0, low_freq_factor=1.0), dict(type='linear', rope_type='yarn', factor=4.0, original_max_position_embeddings=4096)])
def test_options_that_are_not_offered(scaling):
    """What would be dropped in silence makes other tables than the model's."""
    from fla_hip.modules.rotary import rotary_frequencies
    with pytest.raises(ValueError):
        rotary_frequencies(64, scaling=scaling)
    offered = dict(type='yarn', rope_type='yarn', factor=4.0, original_max_position_embeddings=4096, beta_fast=16, beta_slow=2, attention_factor=1.5)
    assert rotary_frequencies(64, scaling=offered)[1] == 1.5


def test_refusals_in_place_come_before_anything_is_written(lib):
    op, both = _mods().rotary_embedding, _mods().rotary_embedding_qk
    cos = torch.ones(8, 8)
    leaf = torch.ones(1, 4, 6, 16, requires_grad=True)
    fused = leaf * 1
    with torch.no_grad():
        quiet = fused[:, :, :2]
    free = torch.ones(1, 4, 2, 16)
    for call in (lambda: op(leaf, cos, cos, inplace=True), lambda: op(leaf[:, :, :2], cos, cos, inplace=True), lambda: op(fused.split([4, 2], 2)[0], cos, cos, inplace=True),
                 lambda: both(*fused.split([4, 2], 2), cos, cos, inplace=True), lambda: both(leaf, free, cos, cos, inplace=True), lambda: both(free, leaf[:, :, 2:], cos, cos, inplace=True),
                 lambda: both(fused[:, :, 2:], leaf[:, :, 2:], cos, cos, inplace=True), lambda: op(quiet, cos, cos, inplace=True)):
        with pytest.raises(RuntimeError, match='inplace=True'):
            call()
    assert not lib.calls and free._version == 0 and fused._version == 0
    q, k = both(fused[:, :, :4], fused[:, :, 4:], cos, cos, inplace=True)
    assert q.requires_grad and k.requires_grad and len(lib.calls) == 2
    q, k = both(free, fused[:, :, 4:], cos, cos, inplace=True)
    assert q is free and not free.requires_grad and free._version == 1 and k.requires_grad and len(lib.calls) == 4


@gpu
@pytest.mark.parametrize('how', ['both', 'queries', 'keys'])
def test_parts_of_one_projection_in_place_under_autograd(how):
    cos, sin = _tables(9, 64)
    x, w = _rows(2, 9, 6, 64, dtype=BF).requires_grad_(), _rows(2, 9, 6, 64, dtype=BF, seed=1)
    other = _rows(2, 9, 2, 64, dtype=BF, seed=2)
    results = []
    for inplace in (False, True):
        fused, free = x * 2, other.clone()
        q, k = (fused[:, :, :4] if how != 'keys' else free), (fused[:, :, 4:] if how != 'queries' else free)
        a, b = _mods().rotary_embedding_qk(q, k, cos, sin, inplace=inplace, seqlen_offsets=torch.zeros(2, dtype=torch.int32, device=DEV))
        whole = torch.cat([a if how != 'keys' else fused[:, :, :4], b if how != 'queries' else fused[:, :, 4:]], 2)
        if inplace:
            assert torch.equal(fused, whole) and (how == 'both' or not free.requires_grad)
        results.append([whole.detach(), a.detach(), b.detach(), *torch.autograd.grad(whole, x, w)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_queries_and_keys_that_overlap(lib):
    """Turned in place at once they would be a race: refused, and only they are - against every element's address."""
    from fla_hip.modules.rotary import overlap
    both, cos = _mods().rotary_embedding_qk, torch.ones(9, 8)
    x = torch.zeros(3, 9, 12, 16, dtype=BF)
    one = x.flatten()
    apart = [(x[:, :, :8], x[:, :, 8:]), (x[:, :, ::2], x[:, :, 1::2]), (x[:1], x[2:]), (x[:, :4], x[:, 4:8]), (x.view(3, 9, 4, 3, 16)[:, :, :, 0], x.view(3, 9, 4, 3, 16)[:, :, :, 2]),
             (one[:640].view(1, 4, 10, 16), one[640:1280].view(1, 4, 10, 16)), (one[:640].view(1, 4, 10, 16), one[640:1024].view(1, 4, 6, 16)), (x.view(3, 9, 6, 32)[..., :16], x.view(3, 9, 6, 32)[..., 16:])]
    meet = [(x[:, :, :8], x[:, :, 7:]), (x[:, :, 3:5], x), (x[:, :8], x[:, 1:]), (x[:, :, ::2], x[:, :, 2::2]), (x, x), (x.view(3, 9, 4, 3, 16)[:, :, :, 0], x[:, :, 9:]),
            (one[:640].view(1, 4, 10, 16), one[639:639 + 384].view(1, 4, 6, 16)), (x[:, 8:], x[:, 8:9, 11:]), (x.view(3, 9, 6, 32)[..., :16], x.view(3, 9, 6, 32)[..., 8:24])]
    for pairs, want in ((apart, False), (meet, True)):
        for q, k in pairs:
            places = [set((t.storage_offset() + sum((torch.arange(n) * s).view(-1, *[1] * (3 - i)) for i, (n, s) in enumerate(zip(t.shape, t.stride())))).flatten().tolist()) for t in (q, k)]
            assert bool(places[0] & places[1]) == overlap(q, k) == overlap(k, q) == want
            if q.shape[:2] != k.shape[:2]:
                continue
            lib.calls.clear()
            if want:
                with pytest.raises(ValueError, match='overlap'):
                    both(q, k, cos, cos, inplace=True)
            else:
                both(q, k, cos, cos, inplace=True)
            assert len(lib.calls) == (not want)
    assert not overlap(x[:, :0], x) and not overlap(x[:, :, :0], x)


def test_positions_of_a_packed_batch_that_the_tables_do_not_have(lib):
    """Where the host has read the boundaries it knows the last position of every sequence."""
    op, x = _mods().rotary_embedding, torch.zeros(1, 7, 2, 16, dtype=BF)
    cu, cos = torch.tensor([0, 2, 7]), torch.zeros(6, 8)
    op(x, cos, cos, cu_seqlens=cu, seqlen_offsets=1)
    op(x, cos[:5], cos[:5], cu_seqlens=cu)
    op(x, cos, cos, cu_seqlens=cu, max_seqlen=5, seqlen_offsets=1)
    for call in (lambda: op(x, cos, cos, cu_seqlens=cu, seqlen_offsets=2), lambda: op(x, cos[:4], cos[:4], cu_seqlens=cu), lambda: op(x, cos, cos, cu_seqlens=cu, seqlen_offsets=-1),
                 lambda: op(x, cos, cos, cu_seqlens=cu, max_seqlen=5, seqlen_offsets=2)):
        with pytest.raises(ValueError, match='positions'):
            call()
    assert len(lib.calls) == 3


def test_tables_do_not_follow_the_modules_type():
    """The buffer of frequencies goes with the module; the tables are formed from those in 64 bits, whatever becomes of it."""
    scaling = dict(type='yarn', factor=4.0, original_max_position_embeddings=64)
    rope, cast = (_mods().RotaryEmbedding(32, scaling=scaling) for _ in range(2))
    cast = cast.half()
    assert cast.inv_freq.dtype == HF and all(torch.equal(a, b) for a, b in zip(rope.tables(300, 'cpu'), cast.tables(300, 'cpu')))
    assert rope.tables(300, 'cpu')[0][0, 0].item() == pytest.approx(rope.attention_factor)


@pytest.mark.parametrize('kw', [dict(), dict(scale_base=512.0, scale_center=10), dict(scaling=dict(type='yarn', factor=4.0, original_max_position_embeddings=64))])
def test_tables_are_made_on_the_host_whatever_the_default_device(kw):
    """Formed on a device by default they would be ready on the stream of that moment only (here: a device that holds no numbers at all)."""
    want = _mods().RotaryEmbedding(32, **kw).tables(50, 'cpu')
    with torch.device('meta'):
        rope = _mods().RotaryEmbedding(32, **kw)
        inside = rope.tables(50, 'cpu')
    assert rope.inv_freq.is_meta and all(torch.equal(a, b) for a, b in zip(want, inside))
