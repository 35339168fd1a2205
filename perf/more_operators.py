"""A step of serving with drafted tokens over a paged cache of keys and values, as cases that can be prepared, run and compared.

Five kinds of work:
  rotary        rotary positions of queries and keys, both layouts, part of a head or all of it: ``rotary_embedding_qk``
  rotary_train  the same with the gradients of both
  append        keys and values of new tokens to their slots in the paged cache, rotated on the way, the queries beside: ``paged_append``
  attn          attention of the new tokens (one, a chain or a tree of drafts) over the paged cache: ``paged_attn``
  keep          the accepted path of a tree moved to the front of the new slots: ``paged_keep``
  verify        which drafted tokens stand against the target's probabilities, from given random numbers: ``verify_drafts``

``own`` false: the plain form, elementary torch operations in 32 bits rounded once at the end (the verification in 64: what decides are values next to
a border).  ``own`` true: the framework's calls.  ``exact`` gives the same results from the definitions in 64 bits."""
import importlib
import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
BYTES = {'bf16': 2, 'f16': 2, 'f32': 4}
MOST_ROTARY = 32768 * 20 * 128          # tokens x heads x features of the largest call
MOST_KEYS = 8 * 32768 * 8 * 128         # sequences x keys x heads x features of the longest caches
MOST_SCORES = 8 * 32 * 32 * 32768       # sequences x rows x heads x keys of the largest call
MOST_VERIFY = 32 * 16 * 131072          # sequences x rows x words


def listed():
    return [
        # A long document's prefill: all of a head in the half layout, positions stretched to four times the trained length.
        dict(name='rotary_prefill', kind='rotary', B=1, T=32768, HQ=16, HK=4, D=128, R=128, interleaved=False, packed=False, stretch=4, dtype='bf16'),
        # A training step that turns a part of each head in the interleaved layout, over a packed batch of documents.
        dict(name='rotary_train', kind='rotary_train', B=1, T=8191, HQ=32, HK=8, D=128, R=64, interleaved=True, packed=True, stretch=1, dtype='f16'),
        # One user's next token on its way into the cache.  Launch and host time.
        dict(name='append_step', kind='append', N=1, S=1, packed=False, HQ=16, HK=4, D=128, R=128, interleaved=False, page=16, context=1000, dtype='bf16'),
        # The prompts of a batch, of all lengths, into pages of 64.
        dict(name='append_prompts', kind='append', N=16, S=2048, packed=True, HQ=32, HK=8, D=128, R=128, interleaved=False, page=64, context=0, dtype='bf16'),
        # One user's next token over a short conversation.
        dict(name='attn_step_1', kind='attn', N=1, S=1, packed=False, tree=False, HQ=16, HK=4, D=128, page=16, context=1000, ragged=False, dtype='bf16'),
        # A batch of conversations of all lengths, a token each.
        dict(name='attn_step_64', kind='attn', N=64, S=1, packed=False, tree=False, HQ=32, HK=8, D=128, page=64, context=8192, ragged=True, dtype='bf16'),
        # Trees of 32 drafted tokens over long documents.
        dict(name='attn_tree_long', kind='attn', N=8, S=32, packed=False, tree=True, HQ=32, HK=8, D=128, page=64, context=32768, ragged=False, dtype='bf16'),
        # Chains of up to 7 drafted tokens in a small odd model with pages of no round size.
        dict(name='attn_chain_odd', kind='attn', N=33, S=7, packed=True, tree=False, HQ=6, HK=3, D=80, page=10, context=3001, ragged=True, dtype='f16'),
        # One user's accepted drafts ...
        dict(name='keep_step', kind='keep', N=1, S=8, HK=4, D=128, page=16, context=1000, dtype='bf16'),
        # ... and those of a batch with large trees.
        dict(name='keep_batch', kind='keep', N=256, S=64, HK=8, D=128, page=64, context=300, dtype='bf16'),
        # Chains of five drafts of a batch at a small vocabulary.
        dict(name='verify_chain', kind='verify', N=16, R=6, V=32000, tree=False, drafted='sampled', dtype='f32'),
        # Trees of 15 sampled drafts at a large vocabulary.
        dict(name='verify_tree', kind='verify', N=32, R=16, V=131072, tree=True, drafted='sampled', dtype='f32'),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    HK = rng.choice([1, 2, 3, 4, 8])
    return HK * rng.choice([1, 2, 3, 4, 8]), HK


def draw(rng):
    kind = rng.choices(['rotary', 'rotary_train', 'append', 'attn', 'keep', 'verify'], [2, 2, 2, 6, 1, 3])[0]
    if kind == 'verify':
        V = rng.choice([32000, 50257, 65536, _log_int(rng, 1000, 131072)])
        R = _log_int(rng, 2, 64)
        return dict(kind=kind, N=_log_int(rng, 1, max(1, min(256, MOST_VERIFY // (R * V)))), R=R, V=V, tree=rng.random() < 0.5,
                    drafted=rng.choice(['sampled', 'given']), dtype=rng.choices(['f32', 'bf16'], [4, 1])[0])
    dtype = rng.choices(['bf16', 'f16'], [3, 1])[0]
    D = rng.choice([64, 128, 128, 256, 8 * rng.randint(5, 32)])
    HQ, HK = _heads(rng)
    page = rng.choice([16, 32, 64, 128, rng.randint(1, 100)])
    if kind == 'keep':
        S = _log_int(rng, 2, 64)
        return dict(kind=kind, N=_log_int(rng, 1, 256), S=S, HK=HK, D=D, page=page, context=_log_int(rng, 1, 1000), dtype=dtype)
    if kind in ('rotary', 'rotary_train', 'append'):
        R, inter = rng.choice([D, D, 2 * rng.randint(1, D // 2)]), rng.random() < 0.4
        if kind == 'append':
            S = _log_int(rng, 1, 4096)
            N = _log_int(rng, 1, max(1, min(256, 32768 * 8 * 128 // (S * HK * D))))
            return dict(kind=kind, N=N, S=S, packed=rng.random() < 0.5, HQ=HQ, HK=HK, D=D, R=R, interleaved=inter, page=page, context=_log_int(rng, 1, 2000), dtype=dtype)
        if rng.random() < 0.2:
            dtype = 'f32'
        B = rng.choice([1, 1, 2, 3, 8])
        T = _log_int(rng, 1 if kind == 'rotary' else 16, MOST_ROTARY // (B * (HQ + HK) * D * (1 if kind == 'rotary' else 2)))
        return dict(kind=kind, B=B, T=min(T, 131072 // B), HQ=HQ, HK=HK, D=D, R=R, interleaved=inter, packed=B == 1 and rng.random() < 0.4, stretch=rng.choice([1, 4]), dtype=dtype)
    S = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 2, 64), _log_int(rng, 16, 256)])
    N = _log_int(rng, 1, 128)
    context = _log_int(rng, 1, max(64, min(131072, MOST_KEYS // (N * HK * D), MOST_SCORES // (N * S * HQ))))
    N = max(1, min(N, MOST_SCORES // (S * HQ * context)))
    return dict(kind=kind, N=N, S=S, packed=rng.random() < 0.4, tree=S > 1 and rng.random() < 0.6, HQ=HQ, HK=HK, D=D, page=page, context=context,
                ragged=rng.random() < 0.5, dtype=dtype)


def _table(positions, R, stretch):
    """cos, sin [positions, R / 2]: frequencies that fall off from 1 to 1/10000, the slow ones stretched for contexts beyond the trained 8192 (those that turn
    less than once in it by the whole factor, those that turn over 32 times not at all)."""
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device='cuda') / R)
    turns = 8192 * inv / (2 * math.pi)
    part = ((turns - 1) / 31).clamp(0, 1)
    inv = inv * (part + (1 - part) / stretch)
    angle = torch.arange(positions, dtype=torch.float64, device='cuda')[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _lengths(case, most, low):
    """Whole numbers from low to most, short ones more often, one for each sequence."""
    return [round(low + (most - low) * ((i + 1) / case['N']) ** 1.5) for i in range(case['N'])]


def _rows(case):
    return _lengths(case, case['S'], 1) if case.get('packed') else [case['S']] * case['N']


def _context(case):
    return _lengths(case, case['context'], 0) if case.get('ragged', case['kind'] == 'append') else [case['context']] * case['N']


def _any_order(gen, lengths):
    return torch.tensor(lengths)[torch.randperm(len(lengths), generator=gen)]


def _pages(case, gen, lengths):
    """(number of pages, table [N, pages of the longest]): the pages of the sequences anywhere in the cache, -1 behind their last."""
    need = (lengths + case['page'] - 1) // case['page']
    # (a cache that holds them in any order of the contexts and new rows)
    total = sum(-(-(c + case['S']) // case['page']) for c in _context(case))
    anywhere = torch.randperm(total, generator=gen)
    first = torch.cumsum(need, 0) - need
    at = torch.arange(int(need.max()))
    table = torch.where(at < need[:, None], anywhere[(first[:, None] + at).clamp(max=total - 1)], -1)
    return total, table.int().cuda()


def _tree(gen, N, R):
    """Parents [N, R] of trees of R rows: row 0 is the root (-1), the others hang on a row before them, nearer ones more often."""
    back = (torch.rand(N, R, generator=gen) ** 2 * torch.arange(R)).floor().long()
    parents = torch.arange(R) - 1 - back.clamp(max=(torch.arange(R) - 1).clamp(min=0))
    parents[:, 0] = -1
    return parents


def _ancestors(parents):
    """[N, R, R] truth values: row i is row j or comes after it."""
    N, R = parents.shape
    sees = torch.zeros(N, R, R, dtype=torch.bool)
    for i in range(R):
        sees[:, i, i] = True
        if i:
            sees[:, i] |= sees[torch.arange(N), parents[:, i]]
    return sees


def _inputs(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device='cuda').to(DTYPES[case['dtype']])
    kind = case['kind']
    if kind == 'verify':
        return _drafts(case, gen, host)
    HK, D = case['HK'], case['D']
    if kind.startswith('rotary'):
        B, T, HQ = case['B'], case['T'], case['HQ']
        t = dict(q=normal(B, T, HQ, D), k=normal(B, T, HK, D))
        if case['packed']:
            # documents of all lengths, their boundaries in the order of the batch
            cut = torch.cat([torch.tensor([0, T]), torch.randint(0, T + 1, (min(T, 11),), generator=host)]).sort().values
            t['cu'] = cut.int().cuda()
        t['cos'], t['sin'] = _table(T + 100, case['R'], case['stretch'])
        if kind == 'rotary_train':
            t['dq'], t['dk'] = normal(B, T, HQ, D), normal(B, T, HK, D)
        return t
    N, S = case['N'], case['S']
    rows = _any_order(host, _rows(case))
    context = _any_order(host, _context(case))
    pages, table = _pages(case, host, context + rows)
    cache = (pages, case['page'], HK, D)
    t = dict(k_cache=normal(*cache), v_cache=normal(*cache), table=table, context=context.int().cuda())
    if case.get('packed'):
        t['cu'] = torch.cat([torch.zeros(1, dtype=torch.long), rows.cumsum(0)]).int().cuda()
    batch = (1, int(rows.sum())) if case.get('packed') else (N, S)
    if kind == 'append':
        t.update(q=normal(*batch, case['HQ'], D), k=normal(*batch, HK, D), v=normal(*batch, HK, D))
        t['cos'], t['sin'] = _table(int((context + rows).max()), case['R'], 1)
    elif kind == 'attn':
        t['q'] = normal(*batch, case['HQ'], D) * 1.5
        if case['tree']:
            sees = _ancestors(_tree(host, N, S))
            if case['packed']:
                sees = torch.cat([s[:int(r)] for s, r in zip(sees, rows)])
            t['mask'] = sees.cuda()
    else:
        # a path down a tree of S rows: the root, then some of the rows behind it, in order
        kept = (1 + torch.rand(N, generator=host) ** 2 * min(S, 8)).long().clamp(max=S)
        path = torch.cat([torch.zeros(N, 1, dtype=torch.long), 1 + torch.rand(N, S - 1, generator=host).argsort(1)], 1)
        path = torch.where(torch.arange(S) < kept[:, None], path, S).sort(1).values
        t['rows'] = torch.where(torch.arange(S) < kept[:, None], path, -1).int().cuda()
        t['kept'] = kept.int().cuda()
    return t


def _drafts(case, gen, host):
    """The target's and the draft's probabilities as two models give them that mostly agree, drafts sampled from the latter (or its first guesses, then
    without probabilities)."""
    N, R, V = case['N'], case['R'], case['V']
    parents = _tree(host, N, R) if case['tree'] else (torch.arange(R) - 1).expand(N, R).contiguous()
    logits = torch.randn(N, R, V, generator=gen, device='cuda') * 3
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits.add_(torch.randn(N, R, V, generator=gen, device='cuda'), alpha=0.7), -1)
    del logits
    up = parents.clamp(min=0).cuda()
    seq = torch.arange(N, device='cuda')[:, None]
    if case['drafted'] == 'sampled':
        many = torch.multinomial(q.view(N * R, V), R, replacement=True, generator=gen).view(N, R, R)
    else:
        many = p.topk(min(R, V), -1).indices
    rank = ((parents[:, :, None] == parents[:, None]) & (torch.arange(R) < torch.arange(R)[:, None])).sum(-1).cuda()
    tokens = many[seq, up, rank].int()
    t = dict(p=p.to(DTYPES[case['dtype']]), tokens=tokens, uniforms=torch.rand(N, R, generator=gen, device='cuda'))
    if case['tree']:
        t['parents'] = parents.int().cuda()
    if case['drafted'] == 'sampled':
        t['q'] = q.to(DTYPES[case['dtype']])
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    if case['kind'] == 'rotary_train':
        t['q'].requires_grad_(True)
        t['k'].requires_grad_(True)
    # (what a server knows without asking the GPU)
    return dict(case=case, longest=case.get('S', case.get('T')), **t)


_calls = None


def _framework():
    global _calls
    if _calls is None:
        importlib.import_module('flash-linear-attention_amd')
        from fla_hip import modules
        from fla_hip.ops import attn, drafts
        _calls = modules, attn, drafts
    return _calls


def run(s):
    train = s['case']['kind'] == 'rotary_train'
    # (inference runs without a graph, as a serving program does)
    with torch.set_grad_enabled(own and train):
        return _run_own(s) if own else PLAIN[s['case']['kind']](s)


def _run_own(s):
    modules, attn, drafts = _framework()
    case = s['case']
    kind = case['kind']
    if kind == 'verify':
        token, accepted, rows = drafts.verify_drafts(s['p'], s['tokens'], s['uniforms'], parents=s.get('parents'), draft_probs=s.get('q'))
        return dict(token=token, accepted=accepted, rows=rows)
    if kind == 'keep':
        attn.paged_keep(s['k_cache'], s['v_cache'], s['table'], s['context'], s['rows'], s['kept'])
        return dict(k_cache=s['k_cache'], v_cache=s['v_cache'])
    if kind == 'append':
        q = attn.paged_append(s['k'], s['v'], s['k_cache'], s['v_cache'], s['table'], s['context'], cu_seqlens=s.get('cu'), max_seqlen=s['longest'],
                              q=s['q'], cos=s['cos'], sin=s['sin'], interleaved=case['interleaved'])
        return dict(q=q, k_cache=s['k_cache'], v_cache=s['v_cache'])
    if kind == 'attn':
        return dict(o=attn.paged_attn(s['q'], s['k_cache'], s['v_cache'], s['table'], s['context'], tree_mask=s.get('mask'), cu_seqlens=s.get('cu'), max_seqlen=s['longest']))
    q, k = modules.rotary_embedding_qk(s['q'], s['k'], s['cos'], s['sin'], interleaved=case['interleaved'], cu_seqlens=s.get('cu'), max_seqlen=s['longest'])
    if kind == 'rotary':
        return dict(q=q, k=k)
    dq, dk = torch.autograd.grad([q, k], [s['q'], s['k']], [s['dq'], s['dk']])
    return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk)


def _turned(x, cos, sin, interleaved):
    """x [..., heads, D], cos and sin [..., R / 2] of the rows' positions."""
    half = cos.shape[-1]
    cos, sin, x32 = cos.unsqueeze(-2), sin.unsqueeze(-2), x.float()
    a, b = (x32[..., 0:2 * half:2], x32[..., 1:2 * half:2]) if interleaved else (x32[..., :half], x32[..., half:2 * half])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x32[..., 2 * half:]], -1).to(x.dtype)


def _places(s, rows):
    """Sequence and place in it of every row of a batch [B, T]."""
    if 'cu' not in s:
        B, T = rows
        return torch.arange(B, device='cuda')[:, None].expand(B, T), torch.arange(T, device='cuda').expand(B, T)
    cu = s['cu'].long()
    at = torch.arange(rows[1], device='cuda')
    seq = torch.searchsorted(cu, at, right=True) - 1
    return seq[None], (at - cu[seq])[None]


def _plain_rotary(s):
    case = s['case']
    _, at = _places(s, (case['B'], case['T']))
    cos, sin = s['cos'][at], s['sin'][at]
    out = {n: _turned(s[n], cos, sin, case['interleaved']) for n in ('q', 'k')}
    if case['kind'] == 'rotary_train':
        out.update({n: _turned(s[n], cos, -sin, case['interleaved']) for n in ('dq', 'dk')})
    return out


def _plain_append(s):
    case = s['case']
    seq, at = _places(s, s['k'].shape[:2])
    at = at + s['context'].long()[seq]
    cos, sin = s['cos'][at], s['sin'][at]
    page, off = s['table'].long()[seq, at // case['page']], at % case['page']
    s['k_cache'][page, off] = _turned(s['k'], cos, sin, case['interleaved'])
    s['v_cache'][page, off] = s['v']
    return dict(q=_turned(s['q'], cos, sin, case['interleaved']), k_cache=s['k_cache'], v_cache=s['v_cache'])


def _plain_attn(s):
    case = s['case']
    N, S, HQ, HK, D, size = case['N'], case['S'], case['HQ'], case['HK'], case['D'], case['page']
    seq, at = _places(s, s['q'].shape[:2])
    q = torch.zeros(N, S, HQ, D, device='cuda')
    q[seq, at] = s['q'].float()
    rows = torch.full((N,), S, device='cuda') if 'cu' not in s else (s['cu'][1:] - s['cu'][:-1]).long()
    context = s['context'].long()
    L = s['table'].shape[1] * size
    key = torch.arange(L, device='cuda')
    page = s['table'].long()[:, key // size].clamp(min=0)
    k, v = (s[c][page, key % size].float().transpose(1, 2) for c in ('k_cache', 'v_cache'))       # [N, HK, L, D]
    new = key - context[:, None]                                                                   # [N, L]
    sees = (new < 0)[:, None] | (new[:, None] <= torch.arange(S, device='cuda')[:, None])          # [N, S, L]
    if 'mask' in s:
        mask = torch.zeros(N, S, S, dtype=torch.bool, device='cuda')
        mask[seq, at] = s['mask'].view(*seq.shape, S)
        sees = (new < 0)[:, None] | mask.gather(2, new.clamp(0, S - 1)[:, None].expand(N, S, L))
    sees = sees & (new < rows[:, None])[:, None]
    scores = q.view(N, S, HK, HQ // HK, D).permute(0, 2, 3, 1, 4).reshape(N, HK, -1, D) @ k.transpose(2, 3) * D ** -0.5
    sees = sees[:, None, None].expand(N, 1, HQ // HK, S, L).reshape(N, 1, -1, L)
    scores = torch.where(sees, scores, -1e30)
    weights = torch.where(sees, torch.exp(scores - scores.max(-1, keepdim=True).values), 0.0)
    o = weights @ torch.where((new < rows[:, None])[:, None, :, None], v, 0.0) / weights.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(N, HK, HQ // HK, S, D).permute(0, 3, 1, 2, 4).reshape(N, S, HQ, D)
    return dict(o=o[seq, at].to(s['q'].dtype))


def _plain_keep(s):
    case = s['case']
    i = torch.arange(case['S'], device='cuda').expand(case['N'], -1)
    on = i < s['kept'][:, None]
    seq = torch.arange(case['N'], device='cuda')[:, None].expand_as(i)[on]
    to, fro = (s['context'][:, None] + i)[on].long(), (s['context'][:, None] + s['rows'])[on].long()
    table, size = s['table'].long(), case['page']
    for c in ('k_cache', 'v_cache'):
        s[c][table[seq, to // size], to % size] = s[c][table[seq, fro // size], fro % size]
    return dict(k_cache=s['k_cache'], v_cache=s['v_cache'])


def _plain_verify(s):
    """Row after row of all sequences at once: a draft that hangs on the row its sequence has come to is taken, or its part of the probabilities is."""
    p, q, tokens, u = s['p'], s.get('q'), s['tokens'].long(), s['uniforms'].double()
    N, R, V = p.shape
    parents = s['parents'].long() if 'parents' in s else (torch.arange(R, device='cuda') - 1).expand(N, R)
    seq = torch.arange(N, device='cuda')
    here, depth = torch.zeros(N, dtype=torch.long, device='cuda'), torch.ones(N, dtype=torch.long, device='cuda')
    rows = torch.full((N, R), -1, dtype=torch.long, device='cuda')
    rows[:, 0] = 0
    left = p[:, 0].double()
    for r in range(1, R):
        word = tokens[:, r]
        drafted = torch.zeros(N, V, dtype=torch.float64, device='cuda').index_put_((seq, word), torch.ones((), dtype=torch.float64, device='cuda')) if q is None else q[seq, here].double()
        asked = parents[:, r] == here
        taken = asked & (u[:, r] * drafted[seq, word] < left[seq, word])
        rest = left * (drafted == 0) if q is None else (left - drafted).clamp(min=0)
        mass = rest.sum(-1, keepdim=True)
        rest = torch.where(mass > 0, rest / mass, left)
        left = torch.where(taken[:, None], p[:, r].double(), torch.where((asked & ~taken)[:, None], rest, left))
        here = torch.where(taken, r, here)
        rows[seq, torch.where(taken, depth, 0)] = torch.where(taken, r, 0)
        depth = depth + taken
    total = left.cumsum(-1)
    token = (total > u[:, :1] * total[:, -1:]).int().argmax(-1)
    return dict(token=token, accepted=depth.int(), rows=rows.int())


PLAIN = dict(rotary=_plain_rotary, rotary_train=_plain_rotary, append=_plain_append, attn=_plain_attn, keep=_plain_keep, verify=_plain_verify)


def _spans(t, N, S):
    """First and last row (exclusive) of every sequence in the flattened batch."""
    cu = t['cu'].tolist() if 'cu' in t else [n * S for n in range(N + 1)]
    return list(zip(cu[:-1], cu[1:]))


def _exact_turn(x, at, case, t, sign=1):
    """The pairs as complex numbers, times cos + i sin."""
    R = case['R']
    z = x.double()
    pair = z[..., :R].unflatten(-1, (R // 2, 2)) if case['interleaved'] else torch.stack([z[..., :R // 2], z[..., R // 2:R]], -1)
    z = z.clone()
    w = torch.view_as_complex(pair.contiguous()) * torch.complex(t['cos'][at].double(), sign * t['sin'][at].double())[:, None]
    w = torch.view_as_real(w)
    z[..., :R] = w.flatten(-2) if case['interleaved'] else w.transpose(-1, -2).flatten(-2)
    return z


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case['kind']
    if kind.startswith('rotary'):
        spans = _spans(t, case['B'], case['T'])
        at = torch.cat([torch.arange(e - b, device='cuda') for b, e in spans])
        turn = lambda n, sign: _exact_turn(t[n].flatten(0, 1), at, case, t, sign).view(t[n].shape)
        return {n: turn(n, -1 if n.startswith('d') else 1) for n in ('q', 'k', 'dq', 'dk') if n in t}
    if kind == 'verify':
        return _exact_verify(case, t)
    k_cache, v_cache = t['k_cache'].double(), t['v_cache'].double()
    table, context, size = t['table'].tolist(), t['context'].tolist(), case['page']
    # the place in the flattened cache of every slot of a sequence
    slots = lambda n, count: (torch.tensor(table[n], device='cuda')[:, None] * size + torch.arange(size, device='cuda')).flatten()[:count]
    if kind == 'keep':
        rows, kept = t['rows'].tolist(), t['kept'].tolist()
        for n in range(case['N']):
            at = slots(n, context[n] + case['S'])
            to, fro = at[context[n]:context[n] + kept[n]], at[[context[n] + r for r in rows[n][:kept[n]]]]
            for c in (k_cache, v_cache):
                c.flatten(0, 1)[to] = c.flatten(0, 1)[fro]
        return dict(k_cache=k_cache, v_cache=v_cache)
    spans = _spans(t, case['N'], case['S'])
    if kind == 'append':
        at = torch.cat([torch.arange(c, c + e - b, device='cuda') for (b, e), c in zip(spans, context)])
        turn = lambda x: _exact_turn(x.flatten(0, 1), at, case, t)
        to = torch.cat([slots(n, context[n] + e - b)[context[n]:] for n, (b, e) in enumerate(spans)])
        k_cache.view(-1, case['HK'], case['D'])[to] = turn(t['k'])
        v_cache.view(-1, case['HK'], case['D'])[to] = t['v'].double().flatten(0, 1)
        return dict(q=turn(t['q']).view(t['q'].shape), k_cache=k_cache, v_cache=v_cache)
    q = t['q'].double().flatten(0, 1)
    o = torch.empty_like(q)
    mask = t['mask'].reshape(-1, case['S']) if 'mask' in t else None
    G = case['HQ'] // case['HK']
    del k_cache, v_cache
    for n, (b, e) in enumerate(spans):
        at = slots(n, context[n] + e - b)
        k, v = (t[c].flatten(0, 1)[at].double() for c in ('k_cache', 'v_cache'))
        hidden = torch.zeros(e - b, len(at), dtype=torch.bool, device='cuda')
        hidden[:, context[n]:] = ~mask[b:e, :e - b] if mask is not None else torch.ones(e - b, e - b, device='cuda').triu(1).bool()
        for h in range(case['HQ']):
            scores = (q[b:e, h] @ k[:, h // G].t().contiguous()) / math.sqrt(case['D'])
            o[b:e, h] = torch.softmax(scores.masked_fill(hidden, -math.inf), -1) @ v[:, h // G]
    return dict(o=o.view(t['q'].shape))


def _exact_verify(case, t):
    """One sequence after the other, by the definition."""
    N, R = case['N'], case['R']
    u, tokens = t['uniforms'].tolist(), t['tokens'].tolist()
    parents = t['parents'].tolist() if 'parents' in t else [[r - 1 for r in range(R)]] * N
    out = dict(token=[], accepted=[], rows=[])
    for n in range(N):
        path = [0]
        left = t['p'][n, 0].double()
        for r in range(1, R):
            if parents[n][r] != path[-1]:
                continue
            word = tokens[n][r]
            chance = 1.0 if 'q' not in t else t['q'][n, path[-1]][word].double()
            if u[n][r] * chance < left[word]:
                path.append(r)
                left = t['p'][n, r].double()
                continue
            rest = left.clone()
            if 'q' in t:
                rest = torch.relu(rest - t['q'][n, path[-1]].double())
            else:
                rest[word] = 0
            if rest.sum() > 0:
                left = rest / rest.sum()
        upto = left.cumsum(0)
        out['token'].append(int((upto <= u[n][0] * upto[-1]).sum()))
        out['accepted'].append(len(path))
        out['rows'].append(path + [-1] * (R - len(path)))
    return {k: torch.tensor(v, device='cuda', dtype=torch.int64 if k == 'token' else torch.int32) for k, v in out.items()}


def work(case):
    kind, b = case['kind'], BYTES[case['dtype']]
    if kind == 'verify':
        # the row that the next word comes from, of the target's probabilities and of the draft's; a word of either for each draft
        N, V, rows = case['N'], case['V'], 2 if case['drafted'] == 'sampled' else 1
        return dict(bytes=N * (V * b * rows + case['R'] * (8 + b * rows)), flops=3 * N * V)
    HK, D = case['HK'], case['D']
    if kind.startswith('rotary'):
        T, half, times = case['B'] * case['T'], case['R'] // 2, 2 if kind.endswith('train') else 1
        return dict(bytes=times * 2 * b * T * (case['HQ'] + HK) * D + case['T'] * half * 8, flops=times * 6 * T * (case['HQ'] + HK) * half)
    N, S = case['N'], case['S']
    if kind == 'keep':
        kept = min(S, 1 + min(S, 8) / 3)
        return dict(bytes=N * kept * 2 * 2 * HK * D * b, flops=0)
    rows, context = sum(_rows(case)), sum(_context(case))
    if kind == 'append':
        half = case['R'] // 2
        return dict(bytes=rows * (2 * b * (case['HQ'] + 2 * HK) * D + half * 8), flops=rows * 6 * (case['HQ'] + HK) * half)
    # (rows and contexts meet in any order: a row of the mean number sees a context of the mean length, and half of the new rows)
    return dict(bytes=2 * b * HK * D * (context + rows) + 2 * b * rows * case['HQ'] * D, flops=4 * rows * case['HQ'] * D * (context + rows / 2) / N)
