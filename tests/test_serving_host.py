"""The serving step's calls on the native host path and on the Python path behind it: the same results, and the same refusals; calls that cannot be finished."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from paged_inputs import DEV, cache, pages_for, table

gpu = pytest.mark.gpu
BF = torch.bfloat16


def _rows(*shape, dtype=BF, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _tables(positions, R):
    t = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return t.cos().float().to(DEV), t.sin().float().to(DEV)


def _rotary(**kw):
    from fla_hip.modules import rotary_embedding, rotary_embedding_qk
    q, k = _rows(1, 9, 4, 64), _rows(1, 9, 2, 64, seed=1)
    cos, sin = _tables(30, 64)
    both = rotary_embedding_qk(q, k, cos, sin, **kw)
    return [*both, rotary_embedding(q, cos, sin, **kw)]


def _train(**kw):
    from fla_hip.modules import rotary_embedding, rotary_embedding_qk
    q, k = _rows(1, 9, 4, 64).requires_grad_(), _rows(1, 9, 2, 64, seed=1).requires_grad_()
    cos, sin = _tables(30, 64)
    a, b = rotary_embedding_qk(q, k, cos, sin, **kw)
    one = rotary_embedding(q, cos, sin, **kw)
    (da,) = torch.autograd.grad(a, q, q, create_graph=True)
    (dda,) = torch.autograd.grad(da, q, q, retain_graph=True)
    return [x.detach() for x in (a, b, one, da, dda, *torch.autograd.grad([a, b, one], [q, k], [a, b, one]))]


def _step(cu=None, **kw):
    from fla_hip.ops.attn import paged_append, paged_attn, paged_keep
    contexts, rows = [40, 0, 17], 3
    kc, vc = cache(pages_for([50] * 3, 16), 16, 2, 64, BF)
    t, context = table([50] * 3, 16, kc.shape[0]).to(DEV), torch.tensor(contexts, dtype=torch.int32, device=DEV)
    shape = (3, rows) if cu is None else (1, 3 * rows)
    q, k, v = _rows(*shape, 4, 64), _rows(*shape, 2, 64, seed=1), _rows(*shape, 2, 64, seed=2)
    cos, sin = _tables(60, 64)
    call = {} if cu is None else dict(cu_seqlens=cu.to(DEV), max_seqlen=rows)
    q2 = paged_append(k, v, kc, vc, t, context, q=q, cos=cos, sin=sin, **call)
    o = paged_attn(q2, kc, vc, t, context, tree_mask=kw.get('mask'), scale=kw.get('scale'), **call)
    none = paged_append(k, v, kc, vc, t, context, **call)
    assert none is None
    assert paged_keep(kc, vc, t, context, torch.tensor([[0, 2, -1]] * 3, dtype=torch.int32, device=DEV), torch.tensor([2, 1, 2], dtype=torch.int32, device=DEV)) is None
    return [q2, o, kc, vc]


def _drafts(**kw):
    from fla_hip.ops.drafts import verify_drafts
    p = torch.softmax(_rows(3, 4, 50, dtype=torch.float32), -1)
    tokens = torch.arange(12, dtype=kw.get('index', torch.int32), device=DEV).view(3, 4)
    u = torch.rand(3, 4, generator=torch.Generator().manual_seed(1)).to(DEV)
    lengths = torch.tensor([4, 2, 3], dtype=torch.int32, device=DEV) if kw.get('lengths') else None
    return list(verify_drafts(p, tokens, u, parents=kw.get('parents'), draft_probs=p.flip(0) if kw.get('q') else None, lengths=lengths))


CU = torch.tensor([0, 3, 3, 9], dtype=torch.int32)
CALLS = {
    'rotary': lambda: _rotary(), 'rotary_interleaved': lambda: _rotary(interleaved=True, seqlen_offsets=5),
    'rotary_packed': lambda: _rotary(cu_seqlens=CU.to(DEV), max_seqlen=6, seqlen_offsets=torch.tensor([1, 2, 3], device=DEV)),
    'rotary_positions': lambda: _rotary(positions=torch.arange(9, device=DEV).flip(0)[None]),
    'train': lambda: _train(), 'train_packed': lambda: _train(cu_seqlens=CU.to(DEV), max_seqlen=6, interleaved=True),
    'step': lambda: _step(), 'step_packed': lambda: _step(CU), 'step_tree': lambda: _step(mask=torch.eye(3, dtype=torch.bool, device=DEV), scale=0.3),
    'step_trees': lambda: _step(mask=torch.eye(3, dtype=torch.bool, device=DEV).expand(3, 3, 3).contiguous(), scale=-1),
    'drafts': lambda: _drafts(), 'drafts_sampled': lambda: _drafts(q=True, lengths=True, index=torch.int64), 'drafts_tree': lambda: _drafts(parents=torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device=DEV)),
}


@gpu
@pytest.mark.parametrize('name', CALLS)
def test_both_host_paths_give_the_same(name, monkeypatch):
    from fla_hip import _lib
    taken = []

    class Watched:
        def __getattr__(self, entry):
            def call(*a):
                out = getattr(host, entry)(*a)
                taken.append(out is not None)
                return out
            return call

    host = _lib.host()
    monkeypatch.setattr(_lib, 'host', Watched)
    native = CALLS[name]()
    assert taken and all(taken), 'not taken by the native path'
    monkeypatch.setattr(_lib, 'host', lambda: _lib._PythonHost)
    python = CALLS[name]()
    assert len(native) == len(python)
    for a, b in zip(native, python):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def _ops():
    """An operand and a call with it, of every operator."""
    from fla_hip.modules import rotary_embedding
    from fla_hip.ops.attn import paged_append, paged_attn, paged_keep
    from fla_hip.ops.drafts import verify_drafts
    kc, vc = cache(4, 16, 2, 64, BF)
    t, context = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV), torch.tensor([3, 0], dtype=torch.int32, device=DEV)
    cos, sin = _tables(30, 64)
    k, q, p = _rows(2, 4, 2, 64), _rows(2, 4, 4, 64), torch.softmax(_rows(2, 3, 50, dtype=torch.float32), -1)
    tokens, u = torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.rand(2, 3, device=DEV)
    rows, kept = torch.tensor([[0, 2], [0, 1]], dtype=torch.int32, device=DEV), torch.tensor([2, 1], dtype=torch.int32, device=DEV)

    def keep(kc):
        paged_keep(kc, vc, t, context, rows, kept)
        return kc

    return {'rotary': (q, lambda q: rotary_embedding(q, cos, sin)), 'append': (k, lambda k: paged_append(k, k, kc, vc, t, context, q=q, cos=cos, sin=sin)),
            'attn': (q, lambda q: paged_attn(q, kc, vc, t, context)), 'keep': (kc, keep), 'verify': (p, lambda p: verify_drafts(p, tokens, u)[2])}


@gpu
@pytest.mark.parametrize('op', ['rotary', 'append', 'attn', 'keep', 'verify'])
@pytest.mark.parametrize('form', ['vmap', 'func_jvp', 'sparse', 'fake'])
def test_tensors_without_plain_memory_raise(op, form):
    x, call = _ops()[op]
    if op == 'verify' and form == 'func_jvp':
        pytest.skip('nothing of it is differentiable')
    want = call(x).clone()
    with pytest.raises(Exception):
        if form == 'vmap':
            torch.vmap(call)(torch.stack([x, x]))
        elif form == 'func_jvp':
            torch.func.jvp(call, (x,), (x,))
        elif form == 'sparse':
            call(x.to_sparse())
        else:
            with FakeTensorMode(allow_non_fake_inputs=True) as mode:
                call(mode.from_tensor(x))
    assert torch.equal(call(x), want)


@gpu
@pytest.mark.parametrize('op', ['rotary', 'append', 'attn', 'verify'])
def test_out_of_memory_can_be_caught(op):
    from fla_hip.modules import rotary_embedding
    from fla_hip.ops.attn import paged_append, paged_attn
    from fla_hip.ops.drafts import verify_drafts
    if op == 'verify':
        p = torch.softmax(_rows(64, 4, 50000, dtype=torch.float32), -1)
        tokens, u = torch.zeros(64, 4, dtype=torch.int32, device=DEV), torch.rand(64, 4, device=DEV)
        call = lambda: verify_drafts(p, tokens, u)[0]
    else:
        kc, vc = cache(600, 16, 2, 64, BF)
        t, context = torch.arange(600, dtype=torch.int32, device=DEV)[None], torch.zeros(1, dtype=torch.int32, device=DEV)
        q, k = _rows(1, 9000, 32, 64), _rows(1, 9000, 2, 64)
        cos, sin = _tables(9000, 64)
        call = {'rotary': lambda: rotary_embedding(q, cos, sin), 'append': lambda: paged_append(k, k, kc, vc, t, context, q=q, cos=cos, sin=sin),
                'attn': lambda: paged_attn(q[:, :200], kc, vc, t, context)}[op]
    want = call()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(1e-9)
    try:
        held = []                                       # (blocks that were reserved before still serve small requests)
        with pytest.raises(torch.OutOfMemoryError):
            for _ in range(20000):
                held.append(call())
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    held.clear()
    assert torch.equal(call(), want)


@gpu
def test_refusals_are_those_of_python():
    from fla_hip.ops.attn import paged_append, paged_attn
    kc, vc = cache(4, 16, 2, 64, BF)
    t, context = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV), torch.tensor([3, 0], dtype=torch.int32, device=DEV)
    q, k = _rows(2, 4, 4, 64), _rows(2, 4, 2, 64)
    for error, call in (
            (ValueError, lambda: paged_attn(q[..., :32], kc, vc, t, context)), (ValueError, lambda: paged_attn(q[:, :, :3], kc, vc, t, context)), (ValueError, lambda: paged_attn(q, kc, vc, t[:1], context)),
            (NotImplementedError, lambda: paged_attn(q.float(), kc.float(), vc.float(), t, context)), (NotImplementedError, lambda: paged_attn(q.clone().requires_grad_(), kc, vc, t, context)),
            (ValueError, lambda: paged_append(k, k[:1], kc, vc, t, context)), (ValueError, lambda: paged_append(k, k, kc, vc.half(), t, context)),
            (ValueError, lambda: paged_attn(q, kc.cpu(), vc, t, context)), (ValueError, lambda: paged_attn(q, kc, vc, t, context.cpu()))):
        with pytest.raises(error):
            call()


@gpu
def test_calls_in_two_threads():
    """The interpreter is free while a call checks and launches."""
    import threading
    ops = _ops()
    want = {name: call(x).clone() for name, (x, call) in ops.items() if name != 'keep'}
    failed = []

    def work(name):
        x, call = ops[name]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(call(x), want[name]):
                    failed.append(name)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(name,)) for name in ('rotary', 'attn', 'verify')]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
