"""Attention of a step's rows over the paged cache (fla_hip.ops.attn.paged_attn) against the 64-bit oracle, element by element.

Tolerance, u = half the spacing of the operands' type relative to it, e = 2^-24, L keys.  A score is a sum of D exact products in fp32 and a scaling: off by (D + 4) e S, S the
largest sum of |q_d k_d| scale; its distance from the maximum and the exponential add 4 e (spread + 1).  So a weight is off by d = 2 ((D + 4) e S + 4 e (spread + 1)) of itself, the sum of the
weights by as much, and for the product with v a weight is rounded once to the operands' type, u.  Both sums have L terms in some order, with the parts' sums rescaled at most
L / 16 times: 2 L e of the sum of the magnitudes A = sum w |v|.  The result is rounded once, u |ref|; a weight below the smallest normal number of fp16 is off by
2^-25 of the largest, of which at most L meet some |v|: L 2^-25 max |v|."""
import pytest
import torch

from oracle import serving_oracle as O
from paged_inputs import DEV, cache, pages_for, table

gpu = pytest.mark.gpu
E = 2.0 ** -24
BF, HF = torch.bfloat16, torch.float16


def _attn():
    from fla_hip.ops import attn
    return attn


def _near(got, ref, size, dots, spread, L, D, v_max):
    assert tuple(got.shape) == tuple(ref.shape)
    got = got.cpu()
    u = torch.finfo(got.dtype).eps / 2
    d = 2 * ((D + 4) * E * dots + 4 * E * (spread + 1))[..., None]
    tol = u * ref.abs() * (1 + 1e-3) + (2 * d + u + 2 * (L + 64) * E) * size + (L * v_max + 1) * (2.0 ** -25 if got.dtype == HF else 2.0 ** -130)
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f'{(err / tol).nan_to_num(nan=1e9).max().item():.2f} of the tolerance'


class Step:
    """A step over a paged cache: tensors on the GPU and what the oracle takes."""

    def __init__(self, contexts, rows, page_size, HQ, HK, D, dtype, packed=False, mask=None, layout='slots', index=torch.int32, seed=0, spoil=None, q_std=1.0, room=0):
        self.contexts, self.rows, self.packed, self.D, self.HQ, self.room = contexts, rows, packed, D, HQ, room
        lengths = [c + r for c, r in zip(contexts, rows)]
        self.L = max(lengths)
        pages = pages_for(lengths, page_size)
        self.k_cache, self.v_cache = cache(pages, page_size, HK, D, dtype, seed, layout)
        self.t = table(lengths, page_size, pages, seed)
        if spoil:
            spoil(self)
        gen = torch.Generator().manual_seed(seed + 77)
        self.firsts = [0, *torch.tensor(rows).cumsum(0).tolist()]
        shape = (1, sum(rows) + room) if packed else (len(rows), rows[0])
        self.q = (torch.randn(*shape, HQ, D, generator=gen) * q_std).to(dtype).to(DEV)
        self.mask = mask                                          # [B,T,cols], [T,cols] or packed [rows,cols], on the CPU
        self.index = index
        self.scale = D ** -0.5

    def call(self, **kw):
        cu = torch.tensor(self.firsts, dtype=self.index, device=DEV) if self.packed else None
        return _attn().paged_attn(kw.pop('q', self.q), self.k_cache, self.v_cache, self.t.to(DEV), torch.tensor(self.contexts, dtype=self.index, device=DEV),
                                  tree_mask=None if self.mask is None else self.mask.to(DEV), cu_seqlens=cu, **kw)

    def sees(self, n, i, j):
        if self.mask is None:
            return j <= i
        row = self.mask[self.firsts[n] + i] if self.packed else self.mask[i] if self.mask.dim() == 2 else self.mask[n, i]
        return j < len(row) and bool(row[j])

    def check(self, o=None, scale=None, **kw):
        o = self.call(scale=scale, **kw) if o is None else o
        spans = list(zip(self.firsts[:-1], self.firsts[1:]))
        ref, size, dots, spread = O.paged_attn(self.q.flatten(0, 1), self.k_cache, self.v_cache, self.t, self.contexts, spans, self.sees, self.scale if scale is None else scale)
        _near(o.flatten(0, 1), ref, size, dots, spread, self.L, self.D, self.v_cache.abs().nan_to_num(0).max().item())
        return o


def _tree(gen, R):
    sees = torch.zeros(R, R, dtype=torch.bool)
    for i in range(R):
        if i:
            sees[i] |= sees[int(torch.randint(0, i, (1,), generator=gen))]
        sees[i, i] = True
    return sees


# head sizes and types, groups of one to many heads, pages from a slot to many
@gpu
@pytest.mark.parametrize(('HQ', 'HK', 'D', 'page_size', 'dtype'), [
    (4, 4, 64, 16, BF), (8, 2, 128, 16, BF), (16, 4, 128, 64, HF), (6, 3, 80, 10, HF), (2, 1, 256, 32, BF), (32, 1, 64, 1, BF), (5, 5, 128, 7, HF), (24, 3, 96, 128, BF), (3, 1, 8, 16, BF), (7, 7, 200, 100, HF),
    (40, 2, 128, 48, BF), (71, 1, 64, 16, HF)])
def test_steps_of_one_token(HQ, HK, D, page_size, dtype):
    Step([0], [1], page_size, HQ, HK, D, dtype).check()
    Step([700, 0, 31, 64, 1, 15], [1] * 6, page_size, HQ, HK, D, dtype, seed=1).check()


@gpu
@pytest.mark.parametrize(('rows', 'HQ', 'HK', 'D', 'page_size', 'dtype'), [
    (2, 4, 4, 64, 16, BF), (8, 8, 2, 128, 16, BF), (17, 8, 8, 128, 64, HF), (33, 4, 2, 80, 10, HF), (64, 8, 1, 128, 32, BF), (100, 3, 1, 256, 16, BF), (130, 8, 2, 64, 5, HF), (31, 2, 2, 128, 1, BF), (70, 5, 5, 40, 64, BF),
    (200, 16, 2, 128, 16, BF)])
@pytest.mark.parametrize('kind', ['chain', 'tree', 'trees', 'packed', 'packed_trees'])
def test_steps_of_many_rows(kind, rows, HQ, HK, D, page_size, dtype):
    gen = torch.Generator().manual_seed(rows)
    contexts, counts = [300, 0, 77], [rows] * 3
    mask = None
    if kind.startswith('packed'):
        counts = [rows, 1, max(1, rows // 3)]
    if kind == 'tree':
        mask = _tree(gen, rows)
    elif kind == 'trees':
        mask = torch.stack([_tree(gen, rows) for _ in range(3)])
    elif kind == 'packed_trees':
        mask = torch.cat([torch.nn.functional.pad(_tree(gen, c), (0, rows - c)) for c in counts])
    step = Step(contexts, counts, page_size, HQ, HK, D, dtype, kind.startswith('packed'), mask, seed=rows)
    step.check()


@gpu
@pytest.mark.parametrize('D', [64, 128, 256])
@pytest.mark.parametrize('packed', [False, True])
def test_long_contexts_of_all_lengths(packed, D):
    """Long enough for a sequence's keys to be shared out, and some that are too short for it."""
    contexts = [20000, 3, 0, 900, 5111, 64]
    Step(contexts, [1] * 6, 64, 4, 2, D, BF, packed, seed=3).check()
    Step(contexts[:3], [3] * 3, 16, 8, 2, D, HF, packed, seed=4).check()


@gpu
@pytest.mark.parametrize('N', [2, 63, 64, 65, 255, 256, 257, 700])
@pytest.mark.parametrize('packed', [False, True])
def test_many_sequences(N, packed):
    """The work is shared out over the sequences by a wave, by a workgroup, in several turns of it; some of them have nothing to do."""
    contexts = [(i * 37) % 150 if i % 5 else 0 for i in range(N)]
    contexts[N // 2] = 2500
    rows = [(i * 7) % 4 for i in range(N)] if packed else [1] * N
    Step(contexts, rows, 16, 2, 1, 64, BF, packed, seed=N).check()


@gpu
@pytest.mark.parametrize('rows', [1, 5, 40])
def test_every_length_around_the_tiles(rows):
    """Contexts and pages that end anywhere inside a tile of keys."""
    contexts = list(range(0, 70)) + [127, 128, 129, 255, 256, 257]
    for page_size in (16, 24, 9):
        Step(contexts, [rows] * len(contexts), page_size, 4, 2, 64, BF, seed=page_size).check()


@gpu
@pytest.mark.parametrize('rows', [3, 40])
def test_rows_that_see_nothing_and_columns_that_are_missing(rows):
    mask = torch.zeros(3, rows, rows, dtype=torch.bool)
    mask[0, 1, 0] = True
    mask[1] = _tree(torch.Generator().manual_seed(0), rows)
    step = Step([0, 0, 5], [rows] * 3, 16, 4, 2, 64, BF, mask=mask)
    o = step.check()
    assert not o[0, 0].any() and not o[0, 2:].any() and o[2].any()
    Step([0, 9, 33], [rows] * 3, 16, 4, 2, 64, BF, mask=mask[:, :, :2]).check()
    wide = torch.ones(rows, rows + 50, dtype=torch.bool)         # (columns behind the rows: nothing there)
    Step([0, 9, 33], [rows] * 3, 16, 4, 2, 64, BF, mask=wide).check()
    inner = torch.zeros(rows, 3, rows, 2, dtype=torch.bool)       # (a mask with strides of its own)
    inner[..., 1] = mask.transpose(0, 1)
    want = step.call()
    step.mask = inner.transpose(0, 1)[..., 1]
    assert torch.equal(step.call(), want)


@gpu
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
@pytest.mark.parametrize(('rows', 'page_size', 'D'), [(1, 16, 64), (6, 16, 128), (6, 10, 128), (40, 64, 128), (80, 7, 64), (24, 16, 256)])
def test_numbers_in_masked_places(rows, page_size, D, bad):
    """NaN and infinities in slots that no row sees - behind the last, in pages of nobody - and in drafts that some rows do not see."""
    contexts = [50, 0, 33]
    gen = torch.Generator().manual_seed(1)
    for mask in (None, torch.stack([_tree(gen, rows) for _ in range(3)])):
        def spoil(step):
            used = torch.zeros(step.k_cache.shape[:2], dtype=torch.bool)
            for n, c in enumerate(contexts):
                for j in range(c + rows):
                    used[O.slot_of(step.t, n, j, *step.k_cache.shape[:2])] = True
            for c in (step.k_cache, step.v_cache):
                c[~used.to(DEV)] = bad
            step.clean = step.k_cache.clone(), step.v_cache.clone()

        step = Step(contexts, [rows] * 3, page_size, 4, 2, D, BF, mask=mask, spoil=spoil)
        step.check()
        # a draft that is not a number: the rows that do not see it get what they got, bit for bit
        want = step.call()
        j = rows // 2
        for cache in (step.k_cache, step.v_cache):
            cache[O.slot_of(step.t, 0, contexts[0] + j, *cache.shape[:2])] = bad
        got = step.call()
        blind = torch.tensor([not step.sees(0, i, j) for i in range(rows)])
        assert torch.equal(got[0, blind], want[0, blind]) and torch.equal(got[1:], want[1:])
        if bad != bad:
            assert got[0, ~blind].isnan().all()
        # ... and one whose key is a number while its value is not: the element of the value that is not a number, in the rows that see it
        step.k_cache.copy_(step.clean[0]), step.v_cache.copy_(step.clean[1])
        step.v_cache[O.slot_of(step.t, 0, contexts[0] + j, *cache.shape[:2])][:, 3] = bad
        got = step.call()
        assert torch.equal(got[0, blind], want[0, blind]) and torch.equal(got[0, :, :, 4:], want[0, :, :, 4:])
        seen = got[0, ~blind][..., 3].float()
        assert seen.isnan().all() if bad != bad else (seen == bad).all()


@gpu
def test_scores_of_any_size():
    """Scores that overflow an exponential without the maximum, all keys alike, a single key, scale zero and negative."""
    Step([300, 2], [4, 4], 16, 4, 2, 128, BF, q_std=300.0).check()
    step = Step([300, 2], [4, 4], 16, 4, 2, 128, BF)
    for scale in (0.0, -0.3, 3.0, 1e-6):
        step.check(scale=scale)
    step.k_cache[:] = step.k_cache[:1, :1]
    step.check()


@gpu
@pytest.mark.parametrize('layout', ['heads', 'one', 'odd'])
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
@pytest.mark.parametrize('rows', [1, 50])
def test_layouts_and_strides(rows, layout, index):
    step = Step([100, 31], [rows] * 2, 16, 4, 2, 64, BF, layout=layout, index=index)
    want = step.check()
    q = step.q
    wide = torch.zeros(*q.shape[:2], 12, 64, dtype=BF, device=DEV)
    wide[:, :, 4:8] = q
    assert torch.equal(step.call(q=wide[:, :, 4:8]), want)
    assert torch.equal(step.call(q=q.transpose(1, 2).contiguous().transpose(1, 2)), want)
    assert torch.equal(step.call(q=torch.cat([q.new_zeros(1), q.flatten()])[1:].view(q.shape)), want)
    assert torch.equal(step.call(q=q.transpose(2, 3).contiguous().transpose(2, 3)), want)
    table = step.t
    step.t = torch.full((2, table.shape[1] + 9), 3, dtype=torch.int64)[:, 4:4 + table.shape[1]].copy_(table)
    assert torch.equal(step.call(), want)


def _no_pages(step):
    step.t[0, 2], step.t[1, 0], step.t[2, 1] = -1, 10 ** 8, -2 ** 31


@gpu
@pytest.mark.parametrize('rows', [1, 30])
@pytest.mark.parametrize('page_size', [16, 5, 64])
def test_keys_without_a_page_are_not_seen(page_size, rows):
    Step([150, 130, 70], [rows] * 3, page_size, 4, 2, 64, BF, spoil=_no_pages).check()
    step = Step([150, 130, 70], [rows] * 3, page_size, 4, 2, 64, BF)
    step.t = step.t[:, :2].clone()                               # (slots behind the table's row)
    step.check()
    step.t = torch.full((3, 4), -1, dtype=torch.int32)
    assert not step.call().any()
    step.t = torch.zeros(3, 0, dtype=torch.int32)
    assert not step.call().any()


@gpu
@pytest.mark.parametrize('rows', [[1, 1, 1], [3, 0, 50], [0, 0, 1], [90, 2, 0]])
def test_packed_batches_with_rows_of_no_sequence(rows):
    step = Step([20, 300, 0], rows, 16, 4, 2, 64, BF, packed=True, room=5)
    for max_seqlen in (None, max(rows), 1, sum(rows) + 5):      # (a hint: the result does not go by it)
        o = step.call(max_seqlen=max_seqlen)
        assert not o[:, sum(rows):].any()
    spans = list(zip(step.firsts[:-1], step.firsts[1:]))
    ref, size, dots, spread = O.paged_attn(step.q[0, :sum(rows)], step.k_cache, step.v_cache, step.t, step.contexts, spans, step.sees, step.scale)
    for max_seqlen in (None, 1):
        _near(step.call(max_seqlen=max_seqlen)[0, :sum(rows)], ref, size, dots, spread, step.L, 64, step.v_cache.abs().max().item())


@gpu
@pytest.mark.parametrize('N', [63, 64, 130])
def test_packed_batches_of_many_sequences(N):
    g = torch.Generator().manual_seed(N)
    contexts, rows = (torch.randint(0, n, (N,), generator=g).tolist() for n in (400, 4))
    step = Step(contexts, rows, 16, 4, 2, 64, BF, packed=True)
    o = step.call(max_seqlen=3)
    spans = list(zip(step.firsts[:-1], step.firsts[1:]))
    ref, size, dots, spread = O.paged_attn(step.q[0, :sum(rows)], step.k_cache, step.v_cache, step.t, step.contexts, spans, step.sees, step.scale)
    _near(o[0, :sum(rows)], ref, size, dots, spread, step.L, 64, step.v_cache.abs().max().item())


@gpu
def test_lengths_that_only_the_gpu_knows():
    """Contexts below zero and beyond the table are held to what is there; boundaries that lead outside of the batch read nothing."""
    step = Step([40, 40], [2, 2], 16, 4, 2, 64, BF)
    want = step.call()
    a = lambda context, cu=None, q=step.q: _attn().paged_attn(q, step.k_cache, step.v_cache, step.t.to(DEV), torch.tensor(context, device=DEV),
                                                             cu_seqlens=None if cu is None else torch.tensor(cu, device=DEV), max_seqlen=None if cu is None else 4)
    got = a([40, 2 ** 40])
    assert torch.equal(got[0], want[0]) and got.isfinite().all()
    got = a([40, -5])
    assert torch.equal(got[0], want[0]) and not got[1].any()
    packed = step.q.view(1, 4, 4, 64)
    for cu in ([0, 2, 2 ** 40], [-7, 2, 4], [0, 9, 4], [0, 2, -1]):
        assert a([40, 40], cu, packed).shape == packed.shape     # (finishes; rows of such sequences are not defined)


@gpu
def test_empty_batches():
    step = Step([40, 40], [2, 2], 16, 4, 2, 64, BF)
    assert step.call(q=step.q[:, :0]).shape == (2, 0, 4, 64)
    none = torch.zeros(0, 3, 4, 64, dtype=BF, device=DEV)
    assert _attn().paged_attn(none, step.k_cache, step.v_cache, step.t[:0].to(DEV), torch.zeros(0, dtype=torch.int32, device=DEV)).shape == none.shape
    o = _attn().paged_attn(step.q, step.k_cache[:0], step.v_cache[:0], step.t.to(DEV), torch.tensor([40, 40], device=DEV))
    assert not o.any()


@gpu
def test_cache_beyond_32_bit_offsets():
    """Pages whose elements lie more than 2^31 elements (and 2^32 bytes) into the cache."""
    page_size, HK, D = 64, 8, 128
    pages = 2 ** 31 // (page_size * HK * D) + 40
    k_cache, v_cache = (torch.zeros(pages, page_size, HK, D, dtype=BF, device=DEV) for _ in range(2))
    small = Step([200, 90], [3, 3], page_size, HK, HK, D, BF)
    far = pages - small.k_cache.shape[0]
    k_cache[far:], v_cache[far:] = small.k_cache, small.v_cache
    want = small.call()
    small.k_cache, small.v_cache, small.t = k_cache, v_cache, torch.where(small.t >= 0, small.t + far, -1).int()
    assert torch.equal(small.call(), want)


@gpu
def test_the_same_call_twice_and_on_another_stream():
    step = Step([5000, 20, 900], [4] * 3, 16, 8, 2, 128, BF)
    want = step.call()
    assert torch.equal(step.call(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [step.call() for _ in range(3)]
    others = [step.call() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs + others)


def _step_call(step, k, v, q, cos, sin, t, context):
    """Append, attend: what an attention layer does in a step."""
    q = _attn().paged_append(k, v, step.k_cache, step.v_cache, t, context, q=q, cos=cos, sin=sin)
    return _attn().paged_attn(q, step.k_cache, step.v_cache, t, context)


@gpu
def test_replayed_graphs_that_share_the_cache():
    step = Step([4000, 20, 900], [2] * 3, 16, 8, 2, 128, BF)
    t, context = step.t.to(DEV), torch.tensor(step.contexts, dtype=torch.int32, device=DEV)
    angle = torch.arange(5000, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-torch.arange(0, 128, 2, device=DEV, dtype=torch.float64) / 128)
    cos, sin = angle.cos().float(), angle.sin().float()
    ins = [[torch.randn(3, 2, h, 128, device=DEV).to(BF) for h in (2, 2, 8)] for _ in range(2)]
    _step_call(step, *ins[0], cos, sin, t, context)
    graphs, outs = [], []
    for k, v, q in ins:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_step_call(step, k, v, q, cos, sin, t, context))
    for turn in range(3):
        context.copy_(torch.tensor([[4000, 20, 900], [3, 4000, 0], [1500, 1, 300]][turn]).clamp(max=torch.tensor(step.contexts)))
        for x in ins[0] + ins[1]:
            x.copy_(torch.randn_like(x.float()))
        for i, g in enumerate(graphs):
            g.replay()
            torch.cuda.synchronize()
            got = outs[i].clone()
            assert torch.equal(got, _step_call(step, *ins[i], cos, sin, t, context))


def _refusals(**sizes):
    """(bytes of a workspace, code) of calls at the C entry, without a workspace: nothing is launched."""
    import ctypes
    from fla_hip import _lib
    lib = _lib.load()
    cache = _lib.PagedCache(k=16, v=16, page_table=16, context=16, pages=2, page_size=4, heads=1, dim=16, table_cols=2, table_stride=2, dtype=0)
    call = _lib.PagedAttnCall(**{**dict(q=16, o=16, B=1, T=1, N=1, HQ=2, max_rows=1), **sizes})
    return lib.gdn_paged_attn_workspace_bytes(ctypes.byref(cache), ctypes.byref(call)), lib.gdn_paged_attn(ctypes.byref(cache), ctypes.byref(call), None, 0, None)


def test_library_refuses_masks_without_columns():
    """A mask of no columns has no place in its rows that could be read."""
    from fla_hip import _lib
    for cols in (0, -1, -2 ** 40):
        assert _refusals(mask=16, mask_cols=cols) == (0, _lib.GDN_ERR_INVALID)
    assert _refusals(mask=16, mask_cols=1)[1] == _refusals(mask_cols=0)[1] == _lib.GDN_ERR_WORKSPACE


def test_library_refuses_more_rows_than_a_launch_has_threads():
    """64 threads for each row of a head, in blocks of 256, below 2^32 in all."""
    from fla_hip import _lib
    for rows in (2 ** 26 - 3, 2 ** 26 - 1):
        assert _refusals(T=rows, HQ=1) == (0, _lib.GDN_ERR_UNSUPPORTED)
    assert _refusals(T=2 ** 26 - 4, HQ=1)[1] == _lib.GDN_ERR_WORKSPACE


@gpu
@pytest.mark.parametrize('sign', [1, -1])
@pytest.mark.parametrize(('rows', 'D', 'page_size'), [(1, 64, 16), (7, 128, 10), (40, 128, 16), (80, 64, 16)])
@pytest.mark.parametrize('dtype', [BF, HF])
def test_scores_beyond_the_steps_of_an_exponent(dtype, rows, D, page_size, sign):
    """Scores so large that their own rounding steps are far above 1: keys that are the same share the weight, wherever the largest score comes, and every other key has
    none.  Equal keys give equal scores in the kernel, so their weights are equal, whatever is lost: the result is the mean of their values, off by its sum in fp32 and the
    rounding of the weights and of the result."""
    context = 200
    first = _attn()
    for large in (3000.0, 60000.0):
        for at in ([0, 1, 150], [199], [40, 170, 171, 172]):
            k = torch.zeros(context + rows, 1, D)
            k[5::7] = -large                                    # (scores far below)
            k[3::7] = 0.5 * large
            k[at] = large
            v = torch.randn(context + rows, 1, D, generator=torch.Generator().manual_seed(rows)).to(dtype)
            pages = -(-(context + rows) // page_size)
            caches = []
            for x in (k, v):
                c = torch.zeros(pages * page_size, 1, D, dtype=dtype)
                c[:context + rows] = x.to(dtype)
                caches.append(c.view(pages, page_size, 1, D).to(DEV))
            q = torch.full((1, rows, 2, D), sign * large, dtype=dtype, device=DEV)
            o = first.paged_attn(q, *caches, torch.arange(pages, dtype=torch.int32, device=DEV)[None], torch.tensor([context], dtype=torch.int32, device=DEV), scale=sign * D ** -0.5)
            want = v[at].double().mean(0)
            tol = torch.finfo(dtype).eps / 2 * (want.abs() * (1 + 1e-3) + v[at].double().abs().mean(0)) + 2 * (context + rows + 64) * E * v[at].double().abs().mean(0) + 2.0 ** -25
            assert bool(((o.cpu().double() - want).abs() <= tol).all()), (large, at, o[0, 0, 0, :4], want[0, :4])


def _one_key_above_many(HQ, HK, D, rows, context, dtype, at, score, value, page_size=64, N=1, bad_at=None, bad=None):
    """N sequences that share the pages of one: the key in slot `at` has score `score` and values `value`, all others score 0 and values from 0.5 to 1.5 (the one in
    slot bad_at: bad).  (o [N, rows, HQ, D], the oracle's, its magnitudes, dots and spread for one sequence)"""
    pages = -(-(context + rows) // page_size)
    gen = torch.Generator().manual_seed(context)
    k = torch.zeros(pages * page_size, HK, D)
    k[at, :, 0] = score
    v = (0.5 + torch.rand(pages * page_size, HK, D, generator=gen)).to(dtype)
    v[at] = value
    if bad is not None:
        v[bad_at, :, 1] = bad
    k_cache, v_cache = (x.to(dtype).view(pages, page_size, HK, D).to(DEV) for x in (k, v))
    q = torch.zeros(N, rows, HQ, D, dtype=dtype, device=DEV)
    q[..., 0] = 1
    order = torch.arange(pages, dtype=torch.int32)
    o = _attn().paged_attn(q, k_cache, v_cache, order.expand(N, pages).contiguous().to(DEV), torch.full((N,), context, dtype=torch.int32, device=DEV), scale=1.0)
    ref = O.paged_attn(q[0, :1], k_cache, v_cache, order[None], [context], [(0, 1)], lambda n, i, j: True, 1.0)
    return o, ref


@gpu
@pytest.mark.parametrize('at', [0, 70000, 131070])
@pytest.mark.parametrize('rows', [1, 9, 40])
@pytest.mark.parametrize('dtype', [BF, HF])
def test_many_small_weights_behind_one_large(dtype, rows, at):
    """131071 keys e^-17.4375 of one key each, whose own values are 0: what is left of the result are the small ones, together 0.35 % of the weights.  A weight is held
    relative to 2^7 times the row's maximum, so one below the smallest normal number of fp16 is off by 2^-32 of the largest: L 2^-32 max |v| in the tolerance that the head
    of this file derives.  (The first row alone is compared: those behind it see a key more each.)"""
    context = 131071
    o, (ref, size, dots, spread) = _one_key_above_many(2, 1, 64, rows, context, dtype, at, 17.4375, 0.0, N=600)
    u, L = torch.finfo(dtype).eps / 2, context + 1
    d = 2 * (68 * E * dots + 4 * E * (spread + 1))[..., None]
    tol = u * ref.abs() * (1 + 1e-3) + (2 * d + u + 2 * (L + 64) * E) * size + (L * 1.5 + 1) * (2.0 ** -32 if dtype == HF else 2.0 ** -130)
    err = (o[:, :1].cpu().double() - ref).abs()
    assert bool((err <= tol).all()), f'{(err / tol).max().item():.2f} of the tolerance, {(err / ref).max().item():.4f} of the result'


@gpu
@pytest.mark.parametrize('slot', [3, 31, 40, 76, 97, 99])
@pytest.mark.parametrize('rows', [1, 40])
@pytest.mark.parametrize('dtype', [BF, HF])
def test_a_value_that_is_not_a_number_behind_a_small_weight(dtype, rows, slot):
    """Wherever its key lies, in a tile of the context or in the last, beside the one that outweighs it - all rows see both - an element that is NaN makes the rows' NaN, and an infinity leaves no number."""
    for D in (64, 128):
        for bad in (float('nan'), float('inf')):
            o, _ = _one_key_above_many(2, 1, D, rows, 100, dtype, slot // 32 * 32 + 2, 30.0, 1.0, page_size=16, bad_at=slot, bad=bad)
            assert (o[..., 1].isnan() if bad != bad else ~o[..., 1].isfinite()).all() and o[..., 0].isfinite().all() and o[..., 2:].isfinite().all(), (D, bad)


# keys through LDS (more than 32 rows of a head of the cache, pages of whole tiles): parts of a head of 128 and of 256 elements, and fp16
@gpu
@pytest.mark.parametrize(('rows', 'HQ', 'HK', 'D', 'page_size', 'dtype'), [(40, 4, 2, 80, 16, HF), (70, 8, 2, 96, 64, BF), (50, 4, 2, 200, 16, HF), (64, 8, 1, 128, 32, HF), (33, 3, 1, 136, 48, BF),
                                                                          (129, 2, 2, 72, 16, HF), (40, 2, 1, 256, 16, HF), (90, 1, 1, 64, 16, HF), (36, 4, 4, 8, 16, BF)])
@pytest.mark.parametrize('kind', ['chain', 'trees', 'packed'])
def test_keys_through_lds(kind, rows, HQ, HK, D, page_size, dtype):
    gen = torch.Generator().manual_seed(rows)
    counts = [rows, 1, max(1, rows // 3)] if kind == 'packed' else [rows] * 3
    mask = torch.stack([_tree(gen, rows) for _ in range(3)]) if kind == 'trees' else None
    Step([300, 0, 77], counts, page_size, HQ, HK, D, dtype, kind == 'packed', mask, seed=rows).check()


@gpu
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
@pytest.mark.parametrize(('rows', 'page_size', 'D', 'dtype'), [(1, 16, 64, HF), (6, 10, 128, HF), (40, 16, 80, HF), (40, 16, 96, BF), (40, 64, 200, BF), (70, 16, 128, HF), (36, 16, 256, HF), (12, 16, 72, HF)])
def test_numbers_in_masked_places_of_other_heads_and_types(rows, page_size, D, dtype, bad):
    """NaN and infinities in slots that no row sees, and in a draft that some rows do not see: nothing of them in those rows."""
    contexts = [50, 0, 33]
    mask = torch.stack([_tree(torch.Generator().manual_seed(n), rows) for n in range(3)])

    def spoil(step):
        used = torch.zeros(step.k_cache.shape[:2], dtype=torch.bool)
        for n, c in enumerate(contexts):
            for j in range(c + rows):
                used[O.slot_of(step.t, n, j, *step.k_cache.shape[:2])] = True
        for c in (step.k_cache, step.v_cache):
            c[~used.to(DEV)] = bad

    step = Step(contexts, [rows] * 3, page_size, 4, 2, D, dtype, mask=mask, spoil=spoil)
    want = step.check()
    j = rows // 2
    step.v_cache[O.slot_of(step.t, 0, contexts[0] + j, *step.v_cache.shape[:2])][:, 5] = bad
    got = step.call()
    sees = torch.tensor([step.sees(0, i, j) for i in range(rows)])
    assert torch.equal(got[0, ~sees], want[0, ~sees]) and torch.equal(got[1:], want[1:])
    assert torch.equal(got[0, :, :, :5], want[0, :, :, :5]) and torch.equal(got[0, :, :, 6:], want[0, :, :, 6:])
    seen = got[0, sees][..., 5].float()
    assert seen.isnan().all() if bad != bad else (seen == bad).all()


@gpu
@pytest.mark.parametrize(('contexts', 'rows', 'HQ', 'HK', 'D', 'page_size', 'dtype'), [([0, 0, 0], [513, 1, 300], 4, 2, 64, 16, BF), ([5, 0, 130], [513, 1, 300], 4, 2, 64, 16, BF), ([0], [900], 2, 1, 128, 64, HF),
                                                                                      ([0], [700], 2, 1, 80, 10, HF), ([3], [260], 2, 2, 256, 32, BF), ([10, 20, 30, 0], [0, 0, 3, 0], 4, 2, 64, 16, BF)])
def test_whole_prompts(contexts, rows, HQ, HK, D, page_size, dtype):
    """Rows just appended that see each other only, or little besides."""
    Step(contexts, rows, page_size, HQ, HK, D, dtype, packed=True).check()


@gpu
@pytest.mark.parametrize('page_size', [4096, 4095])
def test_pages_longer_than_the_sequences(page_size):
    Step([3000, 1, 4094], [3, 3, 3], page_size, 4, 2, 64, BF).check()


@gpu
@pytest.mark.parametrize('rows', [2, 40])
def test_tensors_that_share_memory(rows):
    """Keys and values as halves of a head's row or as one tensor; sequences that read the same pages; one sequence's queries, length, pages and mask for all."""
    both = torch.randn(12, 16, 2, 128, generator=torch.Generator().manual_seed(0)).to(BF).to(DEV)
    step = Step([60, 60], [rows] * 2, 16, 4, 2, 64, BF)
    step.t = torch.arange(12, dtype=torch.int32).expand(2, 12)
    for step.k_cache, step.v_cache in ((both[..., :64], both[..., 64:]), (both[..., :64], both[..., :64])):
        step.q = step.q[:1].expand(2, rows, 4, 64)
        step.mask = None
        want = step.check()
        step.mask = torch.ones(rows, rows, dtype=torch.bool).tril()
        context, t = torch.tensor([60], dtype=torch.int32, device=DEV).expand(2), torch.arange(12, dtype=torch.int32, device=DEV)[None].expand(2, 12)
        assert torch.equal(_attn().paged_attn(step.q, step.k_cache, step.v_cache, t, context, tree_mask=step.mask.to(DEV).expand(2, rows, rows)), want)
        step.mask = torch.ones(1, rows, dtype=torch.bool).expand(rows, rows)
        step.check()


@gpu
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('rows', [4, 40])
def test_scales_of_any_sign(rows, dtype):
    step = Step([100, 7], [rows] * 2, 16, 4, 2, 128, dtype)
    for scale in (0.0, 4.0, -0.5, -3.0):
        step.check(scale=scale)
