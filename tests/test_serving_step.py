"""Steps of speculative serving as a program runs them, one after the other: drafted tokens through the paged cache's attention, their verification, what stands kept -
against attention and the recurrence over the tokens that stood, from scratch in 64 bits.

Tolerances: queries and keys are rounded once behind their turn (u, twice in a score: off by 2 u S, S the sum of magnitudes of a score, and so 4 u S of a weight), the rest
as tests/test_paged_attn.py derives it; states as the recurrence's own tests have them (relative error 5e-3 of bf16 operands)."""
import pytest
import torch

from oracle import gdn_oracle as G
from paged_inputs import DEV

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
E = 2.0 ** -24


class Model:
    """Everything a layer sees of a token, as functions of the token."""

    def __init__(self, words, HQ, HK, D, seed):
        gen = torch.Generator().manual_seed(seed)
        self.q, self.k, self.v = (torch.randn(words, h, D, generator=gen).to(BF) for h in (HQ, HK, HK))
        self.target = torch.softmax(torch.randn(words, words, generator=gen) * 1.5, -1)
        self.draft = torch.softmax(self.target.log() + 0.5 * torch.randn(words, words, generator=gen), -1)


def _exact(model, tokens, cos, sin):
    """Attention of every token of a sequence over those before it: (o, tolerance)."""
    D = model.q.shape[-1]
    t = torch.tensor(tokens)
    c, s = (x.cpu().double()[:len(tokens), None] for x in (cos, sin))

    def turned(x):
        a, b = x.double().chunk(2, -1)
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    q, k, v = turned(model.q[t]), turned(model.k[t]), model.v[t].double()
    G_ = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G_, 1), v.repeat_interleave(G_, 1)
    scores = torch.einsum('ihd,jhd->hij', q, k) * D ** -0.5
    size = torch.einsum('ihd,jhd->hij', q.abs(), k.abs()).amax(-1) * D ** -0.5
    w = torch.softmax(scores.masked_fill(torch.ones(len(t), len(t)).triu(1).bool(), float('-inf')), -1)
    o, magnitude = torch.einsum('hij,jhd->ihd', w, v), torch.einsum('hij,jhd->ihd', w, v.abs())
    u = 2.0 ** -8
    # (a score is off by 2 u S (1 + u): both operands rounded; a weight and the sum of weights by that each)
    tol = u * o.abs() + (4 * u * 1.02 * size.t()[..., None] + u + 2 * (len(t) + 64) * E) * magnitude + 1e-6
    return o, tol


@pytest.mark.parametrize(('shape', 'sampled'), [('chain', True), ('chain', False), ('tree', True), ('tree', False)])
def test_steps_of_drafted_tokens(shape, sampled):
    from fla_hip.modules import RotaryEmbedding
    from fla_hip.ops.attn import paged_append, paged_attn, paged_keep
    from fla_hip.ops.drafts import verify_drafts
    N, R, words, HQ, HK, D, page_size, steps = 3, 6, 40, 4, 2, 64, 16, 12
    model = Model(words, HQ, HK, D, 1)
    gen = torch.Generator().manual_seed(5 + sampled)
    pages = N * 8
    k_cache, v_cache = (torch.full((pages, page_size, HK, D), float('nan'), dtype=BF, device=DEV) for _ in range(2))
    page_table = torch.randperm(pages, generator=gen).view(N, 8).int().to(DEV)
    context = torch.zeros(N, dtype=torch.int32, device=DEV)
    cos, sin = RotaryEmbedding(D).tables(page_size * 8, DEV)
    parents = torch.arange(R) - 1 if shape == 'chain' else torch.tensor([-1, 0, 0, 1, 1, 2])
    depth = torch.zeros(R, dtype=torch.int32)
    sees = torch.eye(R, dtype=torch.bool)
    for r in range(1, R):
        depth[r] = depth[parents[r]] + 1
        sees[r] |= sees[parents[r]]
    depth, tree_mask, on_gpu = depth.to(DEV), sees.to(DEV), parents.int().to(DEV)
    stood = [[] for _ in range(N)]                               # the tokens that stand, and what attention gave for them
    outs = [[] for _ in range(N)]
    root = torch.randint(0, words, (N,), generator=gen)
    stands = 0
    for step in range(steps):
        tokens = torch.zeros(N, R, dtype=torch.long)
        tokens[:, 0] = root
        for r in range(1, R):
            of = model.draft[tokens[:, parents[r]]]
            tokens[:, r] = torch.multinomial(of, 1, generator=gen)[:, 0] if sampled else of.topk(R).indices[:, int((parents[1:r] == parents[r]).sum())]
        q, k, v = (x[tokens].to(DEV) for x in (model.q, model.k, model.v))
        q = paged_append(k, v, k_cache, v_cache, page_table, context, q=q, cos=cos, sin=sin, positions=context[:, None] + depth)
        o = paged_attn(q, k_cache, v_cache, page_table, context, tree_mask=tree_mask)
        token, accepted, rows = verify_drafts(model.target[tokens].to(DEV), tokens.to(DEV), torch.rand(N, R, generator=gen).to(DEV), parents=on_gpu,
                                              draft_probs=model.draft[tokens].to(DEV) if sampled else None)
        paged_keep(k_cache, v_cache, page_table, context, rows, accepted)
        context += accepted
        for n in range(N):
            path = rows[n, :int(accepted[n])].tolist()
            assert path[0] == 0 and all(parents[b] == a for a, b in zip(path, path[1:]))
            stood[n] += tokens[n, path].tolist()
            outs[n] += list(o[n, path].cpu())
            stands += len(path) - 1
        root = token.cpu()
        assert ((root >= 0) & (root < words)).all()
    assert stands >= 5                                           # (drafts do stand, or nothing is tested)
    for n in range(N):
        want, tol = _exact(model, stood[n], cos, sin)
        got = torch.stack(outs[n]).double()
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


def test_the_count_of_drafts_that_stand_is_the_recurrences():
    """The other layers of such a model: a state per drafted token, and `num_accepted_tokens` says which of the last step's is the one to start from."""
    from fla_hip.ops.drafts import verify_drafts
    from fla_hip.ops.gated_delta_rule import fused_recurrent_gated_delta_rule
    N, R, words, H, D, steps = 3, 4, 30, 2, 64, 8
    gen = torch.Generator().manual_seed(3)
    model = Model(words, H, H, D, 2)
    model.q, model.k = (torch.nn.functional.normalize(x.float(), dim=-1).to(BF) for x in (model.q, model.k))
    g, beta = -torch.rand(words, H, generator=gen) * 0.3, torch.rand(words, H, generator=gen)
    pool = torch.zeros(N * R + 2, H, D, D, device=DEV)
    slots = (torch.randperm(N * R, generator=gen) + 1).view(N, R).int().to(DEV)
    accepted = torch.ones(N, dtype=torch.int32, device=DEV)
    stood = [[] for _ in range(N)]
    root = torch.randint(0, words, (N,), generator=gen)
    for step in range(steps):
        tokens = torch.zeros(N, R, dtype=torch.long)
        tokens[:, 0] = root
        for r in range(1, R):
            tokens[:, r] = torch.multinomial(model.draft[tokens[:, r - 1]], 1, generator=gen)[:, 0]
        of = lambda x: x[tokens].to(DEV)
        fused_recurrent_gated_delta_rule(of(model.q), of(model.k), of(model.v), of(g), beta=of(beta), initial_state=pool, output_final_state=True, inplace_final_state=True,
                                         ssm_state_indices=slots, num_accepted_tokens=accepted)
        token, accepted, rows = verify_drafts(of(model.target), tokens.to(DEV), torch.rand(N, R, generator=gen).to(DEV), draft_probs=of(model.draft))
        for n in range(N):
            assert rows[n, :int(accepted[n])].tolist() == list(range(int(accepted[n])))
            stood[n] += tokens[n, :int(accepted[n])].tolist()
        root = token.cpu()
    assert sum(len(s) for s in stood) > N * steps + 5
    for n in range(N):
        t = torch.tensor(stood[n])[None]
        _, want = G.recurrent_gated_delta_rule(model.q[t], model.k[t], model.v[t], g[t], beta[t], None, torch.zeros(1, H, D, D), True)
        got = pool[slots[n, int(accepted[n]) - 1]]
        assert G.get_err_ratio(want[0], got.cpu()) < 5e-3


def test_a_captured_step_replayed():
    """Append, attention, verification and keep in one graph, the lengths counted on inside of it, against the same steps made eagerly on a second cache."""
    from fla_hip.modules import RotaryEmbedding
    from fla_hip.ops.attn import paged_append, paged_attn, paged_keep
    from fla_hip.ops.drafts import verify_drafts
    N, R, words, HQ, HK, D = 2, 5, 5000, 4, 2, 64
    gen = torch.Generator().manual_seed(9)
    parents, depth = torch.tensor([-1, 0, 0, 1, 2], dtype=torch.int32, device=DEV), torch.tensor([0, 1, 1, 2, 2], dtype=torch.int32, device=DEV)
    mask = torch.eye(R, dtype=torch.bool)
    mask[:, 0] = mask[3, 1] = mask[4, 2] = True
    mask = mask.to(DEV)
    cos, sin = RotaryEmbedding(D).tables(200, DEV)
    page_table = torch.randperm(24, generator=gen).view(N, 12).int().to(DEV)
    inputs = [dict(q=torch.randn(N, R, HQ, D, generator=gen).to(BF), k=torch.randn(N, R, HK, D, generator=gen).to(BF), v=torch.randn(N, R, HK, D, generator=gen).to(BF),
                   p=torch.softmax(torch.randn(N, R, words, generator=gen), -1), d=torch.softmax(torch.randn(N, R, words, generator=gen), -1),
                   tokens=torch.randint(0, words, (N, R), generator=gen).int(), u=torch.rand(N, R, generator=gen) * 0.7) for _ in range(5)]

    def step(x, kc, vc, context):
        q = paged_append(x['k'], x['v'], kc, vc, page_table, context, q=x['q'], cos=cos, sin=sin, positions=context[:, None] + depth)
        o = paged_attn(q, kc, vc, page_table, context, tree_mask=mask)
        token, accepted, rows = verify_drafts(x['p'], x['tokens'], x['u'], parents=parents, draft_probs=x['d'])
        paged_keep(kc, vc, page_table, context, rows, accepted)
        context.add_(accepted)
        return o, token, accepted, rows

    state = lambda: [torch.zeros(24, 16, HK, D, dtype=BF, device=DEV), torch.zeros(24, 16, HK, D, dtype=BF, device=DEV), torch.zeros(N, dtype=torch.int32, device=DEV)]
    mine, theirs = state(), state()
    held = {k: v.to(DEV) for k, v in inputs[0].items()}
    step(held, *state())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held, *mine)
    for t in mine:
        t.zero_()
    for x in inputs:
        for k, v in x.items():
            held[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = step(held, *theirs)
        assert all(torch.equal(a, b) for a, b in zip((*outs, *mine), (*want, *theirs)))
    assert (theirs[2] >= len(inputs)).all()
