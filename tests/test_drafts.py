"""Verification of drafted tokens (fla_hip.ops.drafts.verify_drafts): whole numbers, equal to those of the 64-bit oracle.  Inputs are given in fp32 or less and everything that
decides is formed in 64 bits on both sides, in another order of sums: a decision can differ where a number lies within some 1e-13 of a border, which random inputs do not
come near (a hundred thousand words: one in 1e8); borders that are tested are of numbers whose sums are exact."""
import pytest
import torch

from oracle import serving_oracle as O

gpu = pytest.mark.gpu
DEV = 'cuda'
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _verify(*a, **kw):
    from fla_hip.ops.drafts import verify_drafts
    return verify_drafts(*a, **kw)


def _same(p, tokens, u, parents=None, q=None, lengths=None, **kw):
    on = lambda x: None if x is None else x.to(DEV)
    got = _verify(on(p), on(tokens), on(u), parents=on(parents), draft_probs=on(q), lengths=on(lengths))
    want = O.verify_drafts(p, tokens, u, parents, q, lengths)
    for name, a, b in zip(('token', 'accepted', 'rows'), got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b), (name, a.cpu(), b)
    return want


def _trees(N, R, seed):
    gen = torch.Generator().manual_seed(seed)
    parents = torch.full((N, R), -1)
    for r in range(1, R):
        parents[:, r] = (torch.rand(N, generator=gen) * r * 0.999).long() if r % 3 else torch.clamp(r - 1 - (torch.rand(N, generator=gen) * 3).long(), min=0)
    return parents.int()


def _inputs(N, R, V, dtype=FP, sampled=True, tree=False, seed=0, apart=0.7):
    gen = torch.Generator().manual_seed(seed * 1000 + V + R)
    logits = torch.randn(N, R, V, generator=gen) * 2
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits + apart * torch.randn(N, R, V, generator=gen), -1)
    parents = _trees(N, R, seed) if tree else None
    up = (parents if tree else (torch.arange(R) - 1).expand(N, R)).long().clamp(min=0)
    of = q[torch.arange(N)[:, None], up]
    tokens = torch.multinomial(of.view(N * R, V), 1, generator=gen).view(N, R) if sampled else of.topk(min(3, V), -1).indices[..., seed % min(3, V)]
    return dict(p=p.to(dtype), tokens=tokens.int(), u=torch.rand(N, R, generator=gen), parents=parents, q=q.to(dtype) if sampled else None)


@gpu
@pytest.mark.parametrize('tree', [False, True])
@pytest.mark.parametrize('sampled', [False, True])
@pytest.mark.parametrize(('N', 'R', 'V'), [(1, 1, 1), (1, 2, 5), (5, 3, 64), (3, 8, 2047), (3, 8, 2048), (3, 8, 2049), (2, 7, 9001), (70, 20, 33), (1, 100, 40), (2, 1024, 10), (2, 6, 50257), (2, 9, 131073), (200, 5, 70001)])
def test_against_the_oracle(N, R, V, sampled, tree):
    for seed in range(3):
        _same(**_inputs(N, R, V, sampled=sampled, tree=tree, seed=seed))


@gpu
@pytest.mark.parametrize('sampled', [False, True])
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('V', [1, 7, 2051, 8195])
def test_types(dtype, sampled, V):
    _same(**_inputs(4, 9, V, dtype, sampled, tree=True))


@gpu
def test_many_refusals_at_one_row():
    """A root with 40 children that all fall: every one of them has a pass of its own."""
    x = _inputs(3, 41, 3000, seed=5, tree=True, apart=2.0)
    x['parents'] = torch.zeros(3, 41, dtype=torch.int32)
    x['u'] = x['u'] * 0.02 + 0.98
    _same(**x)
    x['q'] = None
    x['tokens'] = x['tokens'] % 7                                # (the same word again and again, too)
    _same(**x)


@gpu
@pytest.mark.parametrize('sampled', [False, True])
def test_nothing_and_everything_stands(sampled):
    x = _inputs(2, 6, 500, sampled=sampled)
    everything = dict(x, u=torch.zeros(2, 6))
    assert (_same(**everything)[1] == 6).all()
    x['p'].scatter_(2, x['tokens'][:, 1:].long().unsqueeze(1).expand(2, 6, 5), 0.0)
    assert (_same(**x)[1] == 1).all()


@gpu
def test_borders():
    """Numbers whose sums are exact: u q = p refuses, and the token is the first whose running sum is above, not at, u."""
    p = torch.tensor([[[0.25, 0.0, 0.5, 0.25], [0.5, 0.5, 0.0, 0.0]]])
    q = torch.tensor([[[0.5, 0.25, 0.25, 0.0], [0.25] * 4]])
    for u0, u1 in [(0.0, 0.5), (0.0, 0.5 - 2.0 ** -24), (0.5, 0.5), (0.25, 0.75), (1 - 2.0 ** -24, 0.75), (0.5, 0.0)]:
        for token in range(4):
            tokens = torch.tensor([[0, token]])
            u = torch.tensor([[u0, u1]])
            _same(p, tokens, u, q=q)
            _same(p, tokens, u)
    # a refused word that had everything: p stays
    one = torch.zeros(1, 2, 4)
    one[..., 2] = 1
    assert _same(one, torch.tensor([[0, 2]]), torch.tensor([[0.5, 1.0]]))[0] == 2
    assert _same(one, torch.tensor([[0, 1]]), torch.tensor([[0.5, 0.0]]), q=one)[0] == 2
    # u of 1 and beyond, and NaN: the last word with a chance
    assert _same(p, torch.tensor([[0, 1]]), torch.tensor([[1.0, 0.5]]))[0] == 3
    assert _same(p[:, :1], torch.tensor([[0]]), torch.tensor([[7.0]]))[0] == 3
    assert int(_verify(p[:, :1].to(DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([[float('nan')]], device=DEV))[0]) == 3


@gpu
def test_probabilities_that_are_none():
    x = _inputs(4, 3, 3000)
    nan = float('nan')
    x['p'][0, :, :2500] = nan
    x['p'][1] = 0.0
    x['p'][2, :, 5] = -1.0
    x['q'][2, :, 7] = nan
    x['p'][3, :, 100] = float('inf')
    x['u'][:, 1:] = 1.0
    want = O.verify_drafts(x['p'][:3], x['tokens'][:3], x['u'][:3], None, x['q'][:3])
    token, accepted, _ = _verify(*(x[k].to(DEV) for k in ('p', 'tokens', 'u')), draft_probs=x['q'].to(DEV))
    assert torch.equal(token[:3].cpu(), want[0]) and token[1] == token[3] == -1 and want[0][1] == -1 and torch.equal(accepted[:3].cpu(), want[1])


@gpu
@pytest.mark.parametrize('sampled', [False, True])
def test_drafts_that_are_none(sampled):
    """Words outside the vocabulary, parents that are not before their rows, rows behind a sequence's length."""
    x = _inputs(4, 8, 100, sampled=sampled, tree=True)
    x['parents'] = torch.tensor([[-1, 0, 1, 2, 3, 4, 5, 6], [5, 0, 2, 9, 0, 7, -3, 1], [-1, 0, 0, 0, 2, 2 ** 31 - 1, -2 ** 31, 1], [-1] * 8], dtype=torch.int32)
    x['tokens'][0, 3], x['tokens'][1, 1], x['tokens'][2, 1] = 100, -1, 2 ** 31 - 1
    x['u'] = x['u'] * 0.3
    _same(**x)
    x['tokens'] = x['tokens'].long()
    x['tokens'][0, 3], x['tokens'][2, 1] = 2 ** 32, -2 ** 40
    _same(**x)
    x['parents'] = None
    for lengths in ([1, 2, 8, 5], [0, -4, 100, 3]):
        _same(**x, lengths=torch.tensor(lengths))


@gpu
def test_strides_and_shared_trees():
    x = _inputs(3, 5, 301, tree=True)
    x['parents'] = torch.tensor([-1, 0, 0, 1, 1])
    want = _same(**x)
    p, q = (torch.zeros(5, 3, 2, 307)[:, :, 0, 3:304].to(DEV) for _ in range(2))
    p.copy_(x['p'].transpose(0, 1)), q.copy_(x['q'].transpose(0, 1))
    got = _verify(p.transpose(0, 1), x['tokens'].long().to(DEV), x['u'].double().to(DEV), parents=x['parents'].to(DEV), draft_probs=q.transpose(0, 1))
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    wide = torch.zeros(3, 5, 301, 2, device=DEV)                 # words apart
    wide[..., 1] = x['p'].to(DEV)
    got = _verify(wide[..., 1], x['tokens'].to(DEV), x['u'].to(DEV), parents=x['parents'].to(DEV), draft_probs=x['q'].to(DEV))
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


@gpu
def test_no_sequences():
    token, accepted, rows = _verify(torch.zeros(0, 3, 10, device=DEV), torch.zeros(0, 3, dtype=torch.int32, device=DEV), torch.zeros(0, 3, device=DEV))
    assert token.shape == (0,) and accepted.shape == (0,) and rows.shape == (0, 3)


@gpu
def test_tokens_are_distributed_as_the_targets():
    """20000 sequences of one chain and one tree over 6 words: the first token after the root against the target's probabilities.  A count of probability p is off by 5
    standard deviations, sqrt(p (1 - p) / 20000), once in a million."""
    N, V = 20000, 6
    gen = torch.Generator().manual_seed(3)
    p1, q1 = torch.softmax(torch.randn(4, V, generator=gen), -1), torch.softmax(torch.randn(4, V, generator=gen), -1)
    for parents in (torch.tensor([-1, 0, 1, 2]), torch.tensor([-1, 0, 0, 0])):
        up = parents.clamp(min=0)
        tokens = torch.stack([torch.multinomial(q1[up[r]], N, replacement=True, generator=gen) for r in range(4)], 1)
        u = torch.rand(N, 4, generator=gen)
        for q in (q1, None):
            token, accepted, rows = (x.cpu() for x in _verify(p1.expand(N, 4, V).to(DEV), tokens.to(DEV), u.to(DEV), parents=parents.to(DEV),
                                                              draft_probs=None if q is None else q1.expand(N, 4, V).to(DEV)))
            first = torch.where(accepted > 1, tokens[torch.arange(N), rows[:, 1].long()], token)
            share = torch.bincount(first, minlength=V) / N
            want = p1[0]
            assert ((share - want).abs() <= 5 * (want * (1 - want) / N).sqrt()).all(), (parents, q is None, share, want)


@gpu
def test_replayed_graph_and_two_graphs_in_turn():
    xs = [_inputs(5, 6, 4000, seed=s, tree=True) for s in range(4)]
    held = [{k: v.to(DEV).clone() for k, v in x.items()} for x in xs[:2]]
    call = lambda h: _verify(h['p'], h['tokens'], h['u'], parents=h['parents'], draft_probs=h['q'])
    call(held[0])
    graphs, outs = [], []
    for h in held:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(h))
    for turn in range(3):
        for g, h, o, x in zip(graphs, held, outs, (xs[turn], xs[turn + 1])):
            for k, v in x.items():
                h[k].copy_(v)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for h, o in zip(held, outs):
            assert all(torch.equal(a, b) for a, b in zip(o, call(h)))


class _Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: 0 if name.endswith('bytes') else self.calls.append(name) or 0


def test_refusals(monkeypatch):
    from fla_hip import _lib
    from fla_hip.ops.drafts import verify
    from fla_hip.ops.gated_delta_rule import _common
    lib = _Library()
    monkeypatch.setattr(_lib, 'load', lambda: lib)
    monkeypatch.setattr(_lib, 'host', lambda: _lib._PythonHost)
    monkeypatch.setattr(_common, 'current_device', lambda: None)
    monkeypatch.setattr(_common, 'current_stream_ptr', lambda dev: 0)
    monkeypatch.setattr(verify, 'require_gpu', lambda x, *_: x.device)
    p, t, u = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    call = lambda p=p, t=t, u=u, **kw: _verify(p, t, u, **kw)
    assert call()[2].shape == (2, 3) and lib.calls == ['gdn_verify_drafts']
    for bad in (lambda: call(p=p[0]), lambda: call(p=p[:, :0]), lambda: call(p=p[..., :0]), lambda: call(t=t[:1]), lambda: call(t=u), lambda: call(u=u[:1]), lambda: call(u=t), lambda: call(draft_probs=p[:, :2]),
                lambda: call(draft_probs=p.half()), lambda: call(parents=torch.zeros(2, dtype=torch.int32)), lambda: call(parents=torch.zeros(3, 2, dtype=torch.int32)), lambda: call(parents=u),
                lambda: call(lengths=torch.zeros(3, dtype=torch.int32)), lambda: call(lengths=torch.zeros(2))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        call(p=p.double())
    assert lib.calls == ['gdn_verify_drafts']


def test_library_refuses():
    import ctypes
    from fla_hip import _lib
    lib = _lib.load()
    with pytest.raises(RuntimeError, match='ROCm GPU'):
        _verify(torch.zeros(1, 1, 1), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1))

    def call(**kw):
        c = _lib.DraftsCall(p=16, tokens=16, uniforms=16, next_token=16, accepted=16, rows=16, N=1, R=2, V=100000, p_dtype=2)
        for k, v in kw.items():
            setattr(c, k, v)
        return lib.gdn_verify_drafts(ctypes.byref(c), None, 0, None)

    invalid = [dict(N=-1), dict(R=0), dict(V=0), dict(p=None), dict(tokens=None), dict(uniforms=None), dict(next_token=None), dict(accepted=None), dict(rows=None), dict(q=16, q_dtype=0)]
    assert [call(**kw) for kw in invalid] == [_lib.GDN_ERR_INVALID] * len(invalid)
    unsupported = [dict(R=1025), dict(V=4194305), dict(N=65536), dict(p_dtype=3)]
    assert [call(**kw) for kw in unsupported] == [_lib.GDN_ERR_UNSUPPORTED] * len(unsupported)
    assert call() == _lib.GDN_ERR_WORKSPACE and call(N=0) == _lib.GDN_OK


def _outside(sampled, tree, dtype=torch.int32):
    """Inputs of which every third draft is a word outside the vocabulary, and the same without those rows: rows without a parent."""
    x = _inputs(40, 12, 300, sampled=sampled, tree=tree, apart=2.0, seed=7)
    if not tree:
        x['parents'] = (torch.arange(12) - 1).expand(40, 12).int()
    x['tokens'], x['u'] = x['tokens'].to(dtype), x['u'] * 0.6
    out = torch.rand(40, 12, generator=torch.Generator().manual_seed(1)) < 0.3
    out[:, 0] = False
    without = dict(x, parents=torch.where(out, -1, x['parents']).int())
    x['tokens'] = torch.where(out, torch.tensor([-1, 300, 2 ** 31 - 1])[torch.arange(12) % 3].to(dtype), x['tokens'])
    return x, without


@pytest.mark.parametrize('tree', [False, True])
@pytest.mark.parametrize('sampled', [False, True])
def test_oracle_of_drafts_outside_the_vocabulary(sampled, tree):
    """They were drawn from nothing, so they take nothing: the oracle says what it says without their rows."""
    x, without = _outside(sampled, tree)
    for a, b in zip(*(O.verify_drafts(d['p'], d['tokens'], d['u'], d['parents'], d['q']) for d in (x, without))):
        assert torch.equal(a, b)
    p, q = torch.tensor([0.5, 0.3, 0.2]), torch.tensor([0.2, 0.3, 0.5])
    u = torch.stack([torch.linspace(0, 1, 1001)[:-1], torch.full((1000,), 0.5)], 1)
    token = O.verify_drafts(p.expand(1000, 2, 3), torch.tensor([[0, -1]]).expand(1000, 2), u, None, q.expand(1000, 2, 3) if sampled else None)[0]
    assert ((torch.bincount(token, minlength=3) / 1000 - p).abs() <= 1.5e-3).all()      # (a thousand equal steps: an end of each word off by one)


@gpu
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
@pytest.mark.parametrize('tree', [False, True])
@pytest.mark.parametrize('sampled', [False, True])
def test_drafts_outside_the_vocabulary_take_nothing(sampled, tree, index):
    x, without = _outside(sampled, tree, index)
    want = _same(**without)
    got = _same(**x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_tokens_of_padded_rows_are_distributed_as_the_targets():
    """As test_tokens_are_distributed_as_the_targets, with rows that a server has padded by -1 in most of the sequences."""
    N, V = 20000, 6
    gen = torch.Generator().manual_seed(4)
    p, q = torch.softmax(torch.randn(4, V, generator=gen), -1), torch.softmax(torch.randn(4, V, generator=gen), -1)
    for parents in (torch.tensor([-1, 0, 1, 2]), torch.tensor([-1, 0, 0, 0])):
        up = parents.clamp(min=0)
        tokens = torch.stack([torch.multinomial(q[up[r]], N, replacement=True, generator=gen) for r in range(4)], 1)
        tokens[torch.arange(4) >= torch.randint(1, 5, (N, 1), generator=gen)] = -1
        u = torch.rand(N, 4, generator=gen)
        token, accepted, rows = (x.cpu() for x in _verify(p.expand(N, 4, V).to(DEV), tokens.to(DEV), u.to(DEV), parents=parents.to(DEV), draft_probs=q.expand(N, 4, V).to(DEV)))
        first = torch.where(accepted > 1, tokens[torch.arange(N), rows[:, 1].long().clamp(min=0)], token)
        share = torch.bincount(first, minlength=V) / N
        assert ((share - p[0]).abs() <= 5 * (p[0] * (1 - p[0]) / N).sqrt()).all(), (parents, share, p[0])
