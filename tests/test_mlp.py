"""The gated feed-forward block (fla_hip.modules: gated_mlp, GatedMLP) and its gradients against the 64-bit oracle.

Tolerances, u = half the spacing of bf16 / fp16 relative to a value, e = 2^-24.  Element by element: what is rounded to 16 bits on the way (h; s = act'(g) u and
a = act(g); dg and du) is off by u times itself, the fp32 sums by (n / 8 + 32) e times the sum of the magnitudes of their n terms (8 or 16 terms a matrix
instruction, parts of a contraction one after the other), and g's share of that goes through the activation, whose slope and slope's slope are at
most 1.13.  All of it is carried through the products on magnitudes, and the result is rounded once.  Over a whole result of 4096 values or more: k independent
roundings, each uniform in half a spacing, leave a relative 2-norm of at most sqrt(k / 3) u: k = 2 for y and dwd (h, itself), 3 for the other gradients (s or a;
dg or du; itself).  Results under fp16's smallest normal number are off by half its smallest step, 2^-25, h and the others too."""
import contextlib

import pytest
import torch

from oracle import modules_oracle as M

gpu = pytest.mark.gpu
DEV = 'cuda'
E = 2.0 ** -24
BF, HF = torch.bfloat16, torch.float16
TINY = 2.0 ** -25


def _mods():
    import fla_hip.modules as mods
    return mods


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(M_, D, F, dtype, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed * 7919 + M_ * 31 + D * 7 + F)
    r = lambda std, *s: (torch.randn(*s, generator=gen) * std).to(dtype).to(DEV)
    return dict(x=r(scale, M_, D), wg=r(D ** -0.5, F, D), wu=r(D ** -0.5, F, D), wd=r(F ** -0.5, D, F), dy=r(1.0, M_, D))


def _near(name, got, ref, spread, roundings):
    """|got - ref| <= u |ref| + spread, element by element, and the 2-norms."""
    assert tuple(got.shape) == tuple(ref.shape), (name, got.shape, ref.shape)
    u = _u(got.dtype)
    err = (got.double() - ref).abs()
    tol = u * ref.abs() + (1 + u) * spread + TINY
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1, f'{name}: {worst:.2f} of the tolerance'
    if err.numel() >= 4096 and ref.norm() > 0:
        rel = (err.norm() / ref.norm()).item()
        assert rel <= (roundings / 3) ** 0.5 * u, f'{name}: {rel:.2e}, {rel / u:.2f} u'


def _reference(t, act):
    """The exact results and how far the roundings on the way may take each element."""
    x, wg, wu, wd, dy = (t[k].double() for k in ('x', 'wg', 'wu', 'wd', 'dy'))
    u = _u(t['x'].dtype)
    (n, D), F = x.shape, wg.shape[0]
    sums = lambda k: (k / 8 + 32) * E
    g, up = x @ wg.t(), x @ wu.t()
    a, da = M.gate_activation(g, act)
    h = a * up
    dg_sum, du_sum = sums(D) * (x.abs() @ wg.abs().t()), sums(D) * (x.abs() @ wu.abs().t())
    slope = 1.13
    off_h = slope * dg_sum * up.abs() + a.abs() * du_sum + (u + 8 * E) * h.abs() + TINY
    off_s = slope * dg_sum * up.abs() + da.abs() * du_sum + (u + 8 * E) * (da * up).abs() + TINY
    off_a = slope * dg_sum + (u + 8 * E) * a.abs() + TINY
    out = dict(y=(h @ wd.t(), off_h @ wd.abs().t() + sums(F) * (h.abs() @ wd.abs().t()), 2))
    dh = dy @ wd
    off_dh = sums(D) * (dy.abs() @ wd.abs())
    s = da * up
    dg, du = dh * s, dh * a
    off_dg = off_dh * (s.abs() + off_s) + dh.abs() * off_s + u * dg.abs() + TINY
    off_du = off_dh * (a.abs() + off_a) + dh.abs() * off_a + u * du.abs() + TINY
    out['dx'] = (dg @ wg + du @ wu, off_dg @ wg.abs() + off_du @ wu.abs() + sums(2 * F) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()), 3)
    xt = x.t().contiguous().t()
    for name, d, off in (('dwg', dg, off_dg), ('dwu', du, off_du)):
        dt = d.t().contiguous()
        out[name] = (dt @ xt, off.t().contiguous() @ xt.abs() + sums(n) * (dt.abs() @ xt.abs()), 3)
    dyt = dy.t().contiguous()
    out['dwd'] = (dyt @ h, dyt.abs() @ off_h + sums(n) * (dyt.abs() @ h.abs()), 2)
    return out


def _step(t, act):
    leaves = [t[k].detach().clone().requires_grad_(True) for k in ('x', 'wg', 'wu', 'wd')]
    y = _mods().gated_mlp(*leaves, activation=act)
    return dict(zip(('y', 'dx', 'dwg', 'dwu', 'dwd'), (y.detach(), *torch.autograd.grad(y, leaves, t['dy']))))


def _check(M_, D, F, dtype, act='swish', seed=0, scale=1.0):
    t = _inputs(M_, D, F, dtype, seed, scale)
    got, ref = _step(t, act), _reference(t, act)
    for name in ref:
        assert got[name].dtype == dtype
        _near(name, got[name], *ref[name])
    with torch.no_grad():
        y = _mods().gated_mlp(t['x'], t['wg'], t['wu'], t['wd'], activation=act)
    _near('y', y, *ref['y'])
    return t, got


ACTS = ['swish', 'sigmoid', 'gelu_tanh']

# smallest; one and few rows around the form of up to 16; every kind of tile, whole and ragged; odd widths (padded)
SIZES = [(1, 8, 8), (1, 1, 1), (3, 2, 5), (1, 2048, 512), (4, 256, 1024), (5, 264, 520), (16, 1000, 2048), (17, 1000, 2048), (15, 13, 1001), (33, 72, 40), (64, 64, 64),
         (65, 128, 4096), (100, 2048, 256), (127, 513, 130), (128, 128, 128), (200, 1024, 2816), (255, 250, 999), (256, 256, 256), (257, 264, 264), (300, 1004, 2690),
         (513, 40, 3000), (700, 512, 1400), (1030, 1024, 1024)]


@gpu
@pytest.mark.parametrize(('size', 'dtype', 'act'), [(s, (BF, HF)[i % 2], ACTS[i % 3]) for i, s in enumerate(SIZES)] + [(s, (HF, BF)[i % 2], 'swish') for i, s in enumerate(SIZES)])
def test_against_the_oracle(size, dtype, act):
    _check(*size, dtype, act)


@gpu
@pytest.mark.parametrize('rows', [1, 2, 7, 15, 16, 17, 31, 33, 48, 63, 64, 65, 96, 127, 129, 192, 255, 257])
def test_row_counts(rows):
    _check(rows, 256, 768, BF, seed=rows)


@gpu
@pytest.mark.parametrize(('D', 'F'), [(8, 4096), (4096, 8), (24, 24), (40, 2056), (2056, 72), (56, 88)])
def test_widths(D, F):
    for rows in (9, 70, 400):
        _check(rows, D, F, BF)


@gpu
@pytest.mark.parametrize('size', [(4096, 2048, 1024), (2999, 1004, 2690), (6000, 1024, 2816), (48, 2048, 5632), (333, 2048, 5632), (1000, 2048, 5632), (4000, 2048, 5632),
                                  (20000, 512, 512), (100, 8192, 64), (300, 4096, 200), (40, 64, 8192)])
def test_full_rounds_of_tiles_and_shared_ones(size):
    """As many tiles as fill the chip more than once, or few of a long contraction: the ones that are left over share out theirs, in every product."""
    _check(*size, BF)


@gpu
def test_large_and_small_values():
    for scale in (1e-3, 30.0):
        for act in ACTS:
            _check(40, 128, 256, BF, act, scale=scale)
    # gates far on either side: the activation is its limit
    t = _inputs(20, 64, 64, BF)
    t['x'] = torch.cat([torch.full((10, 64), 1e4, device=DEV), torch.full((10, 64), -1e4, device=DEV)]).to(BF)
    t['wg'] = torch.full((64, 64), 1.0, device=DEV).to(BF)
    for act in ACTS:
        got, ref = _step(t, act), _reference(t, act)
        for name in ref:
            assert got[name].isfinite().all(), (act, name)
            _near(name, got[name], *ref[name])


@gpu
@pytest.mark.parametrize('rows', [5, 48, 300])
def test_rows_that_are_not_finite_stay_alone(rows):
    mods = _mods()
    t = _inputs(rows, 264, 520, BF)
    with torch.no_grad():
        y0 = mods.gated_mlp(t['x'], t['wg'], t['wu'], t['wd'])
        x = t['x'].clone()
        x[1, 5] = float('nan'); x[3] = float('inf')
        y = mods.gated_mlp(x, t['wg'], t['wu'], t['wd'])
    keep = torch.ones(rows, dtype=torch.bool); keep[[1, 3]] = False
    assert torch.equal(y[keep], y0[keep]) and y[1].isnan().all() and not y[3].isfinite().any()


@gpu
@pytest.mark.parametrize('rows', [3, 60, 600])
def test_weights_that_are_not_finite_in_one_column(rows):
    """A gradient that is not finite in one row of dy leaves the others' dx alone (contractions end inside stages of zeros, which must not meet it)."""
    t = _inputs(rows, 136, 200, BF)
    got = _step(t, 'swish')
    t['dy'][0, 3] = float('inf')
    bad = _step(t, 'swish')
    assert torch.equal(got['dx'][1:], bad['dx'][1:]) and torch.equal(got['y'], bad['y'])
    assert torch.equal(got['dwd'][:3], bad['dwd'][:3]) and torch.equal(got['dwd'][4:], bad['dwd'][4:])


@gpu
def test_strides_shapes_and_packed_weights():
    mods = _mods()
    t = _inputs(24, 256, 512, BF)
    with torch.no_grad():
        ref = mods.gated_mlp(t['x'], t['wg'], t['wu'], t['wd'])
        packed = torch.cat([t['wg'], t['wu']])                                    # one matrix, its halves as views
        wide = torch.zeros(24, 300, dtype=BF, device=DEV); wide[:, 7:263] = t['x']
        off = torch.zeros(512 * 256 + 1, dtype=BF, device=DEV)[1:].view(512, 256); off.copy_(t['wg'])
        assert torch.equal(mods.gated_mlp(t['x'], packed[:512], packed[512:], t['wd']), ref)
        assert torch.equal(mods.gated_mlp(wide[:, 7:263], t['wg'], t['wu'], t['wd'].t().contiguous().t()), ref)
        assert torch.equal(mods.gated_mlp(t['x'], off, t['wu'], t['wd']), ref)
        assert torch.equal(mods.gated_mlp(t['x'].view(2, 3, 4, 256), t['wg'], t['wu'], t['wd']).view(24, 256), ref)
        assert torch.equal(mods.gated_mlp(t['x'][0], t['wg'], t['wu'], t['wd']), mods.gated_mlp(t['x'][:1], t['wg'], t['wu'], t['wd'])[0])
    a, b = _step(t, 'swish'), _step({**t, 'dy': t['dy'].t().contiguous().t()}, 'swish')
    assert all(torch.equal(a[k], b[k]) for k in a)
    x = t['x'].clone().requires_grad_(True)
    one = torch.autograd.grad(mods.gated_mlp(x, t['wg'], t['wu'], t['wd']).sum(), x)[0]              # an expanded gradient
    two = torch.autograd.grad(mods.gated_mlp(x, t['wg'], t['wu'], t['wd']), x, torch.ones_like(x))[0]
    assert torch.equal(one, two)


@gpu
@pytest.mark.parametrize('size', [(40, 256, 512), (40, 250, 509)])
def test_gradients_that_are_asked_for(size):
    """Every set of inputs that want gradients, by requires_grad and by what autograd asks of one graph; a graph used twice."""
    t = _inputs(*size, BF)
    full = _step(t, 'swish')
    names = ('x', 'wg', 'wu', 'wd')
    for bits in range(1, 16):
        want = [i for i in range(4) if bits >> i & 1]
        leaves = [t[k].clone().requires_grad_(i in want) for i, k in enumerate(names)]
        y = _mods().gated_mlp(*leaves)
        for again in range(2):
            got = torch.autograd.grad(y, [leaves[i] for i in want], t['dy'], retain_graph=True)
            assert all(torch.equal(g, full['d' + names[i]]) for g, i in zip(got, want)), (want, again)
        some = want[len(want) // 2]
        assert torch.equal(torch.autograd.grad(y, leaves[some], t['dy'])[0], full['d' + names[some]])


def _unpack(x):
    """Strided, between 16-byte boundaries, in fp32."""
    x = x.to(DEV).float()
    wide = torch.zeros(*x.shape[:-1], x.shape[-1] + 3, device=DEV)
    wide[..., 1:-2] = x
    return wide[..., 1:-2]


@gpu
@pytest.mark.parametrize('path', ['native', 'strided', 'autocast'])
@pytest.mark.parametrize('size', [(40, 256, 512), (40, 250, 509), (7, 64, 96)])
def test_saved_tensors_may_come_back_in_another_layout_type_and_place(path, size):
    """Saved-tensor hooks: every tensor goes to the host and comes back in fp32.  What they hold is the same: so are the gradients' bits."""
    t = _inputs(*size, BF)
    x = t['x']
    if path == 'strided':
        x = torch.zeros(size[0], size[1] + 8, dtype=BF, device=DEV)[:, :size[1]].copy_(x)

    def grads(*hooks):
        leaves = [v.detach().requires_grad_(True) for v in (x, t['wg'], t['wu'], t['wd'])]
        if path == 'autocast':
            leaves = [v.detach().float().requires_grad_(True) for v in leaves]
        with torch.autograd.graph.saved_tensors_hooks(*hooks) if hooks else contextlib.nullcontext():
            with torch.autocast('cuda', dtype=BF, enabled=path == 'autocast'):
                y = _mods().gated_mlp(*leaves)
        return torch.autograd.grad(y, leaves, t['dy'])

    for i, (a, b) in enumerate(zip(grads(), grads(lambda x: x.cpu(), _unpack))):
        assert a.dtype == b.dtype and torch.equal(a, b), i


@gpu
@pytest.mark.parametrize('strided', [False, True])
def test_saved_tensors_of_another_size_are_refused(strided):
    t = _inputs(20, 64, 96, BF)
    x = torch.zeros(20, 64 + 8 * strided, dtype=BF, device=DEV)[:, :64].requires_grad_(True)
    for shape in ((20, 64), (96, 64), (64, 96), (20, 96)):
        leaves = [x, *(t[k].clone().requires_grad_(True) for k in ('wg', 'wu', 'wd'))]
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x[:-1] if x.shape == shape else x):
            y = _mods().gated_mlp(*leaves)
        with pytest.raises(ValueError, match='came back'):
            y.sum().backward()


def test_what_the_library_gets_of_saved_tensors_that_came_back_otherwise(monkeypatch):
    """The host path in Python (CPU: the library keeps record): with hooks that hand back fp32, strided, the kernel is still given 16-bit memory, 16-byte aligned."""
    from fla_hip import _lib
    from fla_hip.modules import mlp

    class Library:
        def __getattr__(self, name):
            return lambda *a: 0

    got = []
    monkeypatch.setattr(_lib, 'load', Library)
    monkeypatch.setattr(mlp, 'require_gpu', lambda x, *_: x.device)
    monkeypatch.setattr(mlp, 'ptr', lambda t: got.append(t))
    monkeypatch.setattr(mlp, 'launch', lambda *a: None)
    x, wg, wu, wd = (torch.randn(*s).to(BF).requires_grad_(True) for s in ((20, 24), (40, 24), (40, 24), (24, 40)))
    unpack = lambda t: torch.stack([t.float(), t.float()], -1)[..., 0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = mlp.GatedMLPFunction.apply(x, wg, wu, wd, _lib.ACT_SILU)
    got.clear()
    y.sum().backward()
    assert len(got) >= 14
    for t in got:
        assert t is None or (t.dtype in (BF, torch.uint8) and t.is_contiguous() and t.data_ptr() % 16 == 0), (t.dtype, t.stride())


@gpu
def test_a_second_derivative_is_refused():
    for D in (64, 60):
        t = _inputs(8, D, 64, BF)
        for x in (t['x'], torch.zeros(8, D + 4, device=DEV, dtype=BF)[:, :D]):    # (native host path; a strided x takes the other one)
            x = x.requires_grad_(True)
            (g,) = torch.autograd.grad(_mods().gated_mlp(x, t['wg'], t['wu'], t['wd']).sum(), x, create_graph=True)
            with pytest.raises(RuntimeError, match='differentiate twice'):
                g.sum().backward()


@gpu
@pytest.mark.parametrize('act', ACTS)
def test_the_gradient_is_the_difference(act):
    """Differences of the 64-bit oracle's forward along a direction for each input (step 1e-4: their own error is far under the gradients' roundings).  A
    gradient is off by at most u in the 2-norm (three roundings), so its product with a unit direction by at most u times its norm."""
    t = _inputs(64, 96, 160, BF)
    got = _step(t, act)
    args = [t[k].double() for k in ('x', 'wg', 'wu', 'wd')]
    for i, name in enumerate(('dx', 'dwg', 'dwu', 'dwd')):
        g = got[name].double()
        gen = torch.Generator().manual_seed(i)
        v = torch.randn(g.shape, generator=gen).double().to(DEV) / g.numel() ** 0.5 + g / g.norm()
        v = v / v.norm()
        f = lambda z: (M.gated_mlp(*args[:i], args[i] + z * v, *args[i + 1:], act) * t['dy'].double()).sum()
        want = (f(1e-4) - f(-1e-4)) / 2e-4
        assert ((g * v).sum() - want).abs() <= _u(BF) * g.norm() + 1e-6 * want.abs(), (name, (g * v).sum(), want)


@gpu
def test_the_same_call_gives_the_same_bits_and_streams_do_not_matter():
    for size in ((9, 512, 1024), (100, 512, 1024), (2000, 512, 1024)):
        t = _inputs(*size, BF)
        a, b = _step(t, 'swish'), _step(t, 'swish')
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c = _step(t, 'swish')
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a[k], b[k]) and torch.equal(a[k], c[k]) for k in a), size


@gpu
def test_two_calls_at_once():
    """Calls on two streams whose contractions are shared out: a workspace each."""
    ts = [_inputs(100, 512, 1024, BF, seed=s) for s in (1, 2)]
    want = [_step(t, 'swish') for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    got = [None, None]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _step(ts[i], 'swish')
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(g[k], w[k]) for k in w)


@gpu
@pytest.mark.parametrize('size', [(1, 256, 512), (100, 256, 512), (700, 256, 512)])
def test_captured_and_replayed(size):
    """Two graphs of a training step, replayed in turn on new inputs with eager work between."""
    ts = [_inputs(*size, BF, seed=s) for s in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(ts[0], 'swish')
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in ts:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(t, 'swish'))
        graphs.append(graph)
    for seed in range(3):
        eager = []
        for i, t in enumerate(ts):
            new = _inputs(*size, BF, seed=10 + 2 * seed + i)
            eager.append(_step(new, 'swish'))
            for k in t:
                t[k].copy_(new[k])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert all(torch.equal(o[k], e[k]) for k in e), seed


@gpu
def test_more_elements_than_32_bits_count():
    """Rows whose inner activations lie beyond 2^32 bytes (and 2^31 elements)."""
    rows, D, F = 300_007, 64, 8192
    t = _inputs(600, D, F, BF)
    x = torch.zeros(rows, D, dtype=BF, device=DEV)
    dy = torch.zeros_like(x)
    x[-600:], dy[-600:] = t['x'], t['dy']
    got = _step({**t, 'x': x, 'dy': dy}, 'swish')
    ref = _reference(t, 'swish')
    for name in ('y', 'dx'):
        _near(name, got[name][-600:], *ref[name])
        assert not got[name][:-600].any()
    for name in ('dwg', 'dwu', 'dwd'):
        _near(name, got[name], ref[name][0], ref[name][1] + rows / 8 * E * ref[name][0].abs(), ref[name][2])


@gpu
def test_no_rows():
    t = _inputs(0, 64, 128, BF)
    got = _step(t, 'swish')
    assert got['y'].shape == got['dx'].shape == (0, 64)
    assert not got['dwg'].any() and not got['dwu'].any() and not got['dwd'].any()


@gpu
@pytest.mark.parametrize('rows', [5, 100, 300])
def test_the_entry_points_write_their_results_only(rows):
    """Through the C ABI into the middle of larger buffers."""
    from fla_hip import _lib
    from fla_hip.ops.gated_delta_rule._common import launch, ptr
    D, F = 136, 264
    t = _inputs(rows, D, F, BF)
    lib, dev = _lib.load(), torch.device('cuda', torch.cuda.current_device())
    big = {}

    def room(name, n, dtype=BF):
        big[name] = torch.full((n + 128,), 7.0 if dtype == BF else 7, dtype=dtype, device=DEV)
        return big[name][64:64 + n]

    y, h, s, a, dg, du = (room(n, rows * w) for n, w in (('y', D), ('h', F), ('s', F), ('a', F), ('dg', F), ('du', F)))
    dx, dwg, dwu, dwd = room('dx', rows * D), room('dwg', F * D), room('dwu', F * D), room('dwd', F * D)
    sizes = [lib.gdn_gated_mlp_workspace_bytes(rows, D, F, b) for b in (0, 1)]
    ws = [room(f'ws{b}', n, torch.uint8) for b, n in enumerate(sizes)]
    launch(lib.gdn_gated_mlp_fwd, dev, ptr(t['x']), ptr(t['wg']), ptr(t['wu']), ptr(t['wd']), ptr(y), ptr(s), ptr(a), ptr(h), ptr(ws[0]), sizes[0], rows, D, F, 1, 0)
    launch(lib.gdn_gated_mlp_bwd, dev, ptr(t['dy']), ptr(t['x']), ptr(t['wg']), ptr(t['wu']), ptr(t['wd']), ptr(s), ptr(a), ptr(h), ptr(dg), ptr(du),
           ptr(dx), ptr(dwg), ptr(dwu), ptr(dwd), ptr(ws[1]), sizes[1], rows, D, F, 0)
    torch.cuda.synchronize()
    ref = _reference(t, 'swish')
    for name, got in (('y', y), ('dx', dx), ('dwg', dwg), ('dwu', dwu), ('dwd', dwd)):
        _near(name, got.view(ref[name][0].shape), *ref[name])
    for name, b in big.items():
        assert (b[:64] == 7).all() and (b[-64:] == 7).all(), name


@gpu
def test_the_layer_and_autocast():
    mods = _mods()
    torch.manual_seed(0)
    mlp = mods.GatedMLP(hidden_size=256, device=DEV)
    assert mlp.intermediate_size == 768 and {n for n, _ in mlp.named_parameters()} == {'gate_proj.weight', 'up_proj.weight', 'down_proj.weight'}
    assert mods.GatedMLP(64, hidden_ratio=2, device=DEV).intermediate_size == 256 and mods.GatedMLP(64, intermediate_size=100, device=DEV).intermediate_size == 100
    x = torch.randn(2, 50, 256, device=DEV)
    with torch.autocast('cuda', dtype=BF):
        y = mlp(x.requires_grad_(True))
    y.float().square().sum().backward()
    low = [p.detach().to(BF) for p in (mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight)]
    with torch.no_grad():
        assert torch.equal(y, mods.gated_mlp(x.to(BF), *low))
    assert y.dtype == BF and x.grad.dtype == torch.float32 and mlp.gate_proj.weight.grad.dtype == torch.float32
    with pytest.raises(NotImplementedError):
        mlp(x)


def _refusals():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)
    return [
        ('an activation', ValueError, lambda f: f(z(4, 8), z(16, 8), z(16, 8), z(8, 16), activation='relu')),
        ('a gate of another width', ValueError, lambda f: f(z(4, 8), z(16, 9), z(16, 8), z(8, 16))),
        ('a gate of one dimension', ValueError, lambda f: f(z(4, 8), z(8), z(16, 8), z(8, 16))),
        ('an up projection of another width', ValueError, lambda f: f(z(4, 8), z(16, 8), z(15, 8), z(8, 16))),
        ('a down projection that is not turned', ValueError, lambda f: f(z(4, 8), z(16, 8), z(16, 8), z(16, 8))),
        ('no inner features', ValueError, lambda f: f(z(4, 8), z(0, 8), z(0, 8), z(8, 0))),
        ('no features', ValueError, lambda f: f(z(4, 0), z(16, 0), z(16, 0), z(0, 16))),
        ('no dimension', ValueError, lambda f: f(z(()), z(16, 1), z(16, 1), z(1, 16))),
        ('two types', ValueError, lambda f: f(z(4, 8), z(16, 8), z(16, 8, dtype=HF), z(8, 16))),
        ('32 bits', NotImplementedError, lambda f: f(*(z(*s, dtype=torch.float32) for s in ((4, 8), (16, 8), (16, 8), (8, 16))))),
    ]


@pytest.mark.parametrize(('what', 'error', 'call'), _refusals(), ids=[r[0] for r in _refusals()])
def test_refusals(what, error, call, monkeypatch):
    from fla_hip.modules import mlp
    monkeypatch.setattr(mlp, 'require_gpu', lambda x, *_: x.device)
    with pytest.raises(error):
        call(mlp.gated_mlp)


def test_cpu_tensors_and_unknown_layers_are_refused():
    z = torch.zeros
    with pytest.raises(RuntimeError, match='GPU'):
        _mods().gated_mlp(z(4, 8, dtype=BF), z(16, 8, dtype=BF), z(16, 8, dtype=BF), z(8, 16, dtype=BF))
    with pytest.raises(ValueError):
        _mods().GatedMLP(64, hidden_act='relu')


def test_the_entry_points_refuse():
    """By the library's host code: nothing is launched."""
    from fla_hip import _lib
    try:
        lib = _lib.load()
    except _lib.GDNLibraryError:
        pytest.skip('not built in this checkout')
    P = 1 << 20                                                                    # (an address that is never read)

    def fwd(M_=300, D=256, F=512, x=P, y=P, h=P, s=None, a=None, ws=P, n=1 << 40, act=1, dt=0):
        return lib.gdn_gated_mlp_fwd(x, P, P, P, y, s, a, h, ws, n, M_, D, F, act, dt, None)

    def bwd(M_=300, D=256, F=512, dy=P, s=P, h=P, dg=P, dx=P, dwg=P, dwd=P, ws=P, n=1 << 40, dt=0):
        return lib.gdn_gated_mlp_bwd(dy, P, P, P, P, s, P, h, dg, P, dx, dwg, P, dwd, ws, n, M_, D, F, dt, None)

    assert fwd(M_=-1) == fwd(D=0) == fwd(x=None) == fwd(y=None) == fwd(h=None) == fwd(s=P) == fwd(x=P + 8) == fwd(h=P + 2) == _lib.GDN_ERR_INVALID
    assert fwd(D=12) == fwd(F=9) == fwd(dt=2) == fwd(act=0) == fwd(act=4) == fwd(D=1 << 21) == fwd(M_=1 << 30) == _lib.GDN_ERR_UNSUPPORTED
    assert lib.gdn_gated_mlp_workspace_bytes(48, 2048, 5632, 0) > 0 and lib.gdn_gated_mlp_workspace_bytes(48, 2048, 5632, 1) > 0 and lib.gdn_gated_mlp_workspace_bytes(16, 256, 512, 0) == 0
    assert fwd(48, 2048, 64, ws=None) == fwd(48, 2048, 64, n=16) == _lib.GDN_ERR_WORKSPACE       # (the first launch already needs it)
    assert fwd(M_=0, x=None) == _lib.GDN_OK
    assert bwd(dy=None) == bwd(s=None) == bwd(h=None) == bwd(dg=None) == bwd(dg=P + 8) == _lib.GDN_ERR_INVALID
    assert bwd(F=12) == bwd(dt=2) == _lib.GDN_ERR_UNSUPPORTED
    assert bwd(48, 2048, 64, ws=None) == _lib.GDN_ERR_WORKSPACE
    assert lib.gdn_gated_mlp_workspace_bytes(-1, 8, 8, 0) == lib.gdn_gated_mlp_workspace_bytes(8, 12, 8, 1) == 0


def test_a_workspace_between_16_byte_boundaries_is_refused():
    """By the library's host code: nothing is launched.  (Up to 16 rows there is none to look at.)"""
    from fla_hip import _lib
    try:
        lib = _lib.load()
    except _lib.GDNLibraryError:
        pytest.skip('not built in this checkout')
    P, n = 1 << 20, 1 << 40
    for off in (4, 8, 12):
        assert lib.gdn_gated_mlp_fwd(*[P] * 5, None, None, P, P + off, n, 48, 2048, 64, 1, 0, None) == _lib.GDN_ERR_INVALID
        assert lib.gdn_gated_mlp_bwd(*[P] * 14, P + off, n, 48, 2048, 64, 0, None) == _lib.GDN_ERR_INVALID


@gpu
def test_matrices_of_other_sizes():
    """gdn_pad_rows: zeros where there is no source, several matrices in a launch, nothing beside them."""
    import ctypes

    from fla_hip import _lib
    from fla_hip.ops.gated_delta_rule._common import launch, ptr

    class Segment(ctypes.Structure):
        _fields_ = [('src', ctypes.c_void_p), ('dst', ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ('src_rows', 'src_cols', 'dst_rows', 'dst_cols')]

    lib, dev = _lib.load(), torch.device('cuda', torch.cuda.current_device())
    sizes = [((5, 7), (8, 8)), ((300, 1001), (300, 1008)), ((16, 24), (13, 19)), ((1, 1), (3, 2))]
    src = [torch.randn(*a, device=DEV).to(BF) for a, _ in sizes]
    dst = [torch.full((b[0] * b[1] + 33,), 7.0, dtype=BF, device=DEV) for _, b in sizes]
    segs = (Segment * 4)(*(Segment(ptr(s), d.data_ptr() + 2, *a, *b) for s, d, (a, b) in zip(src, dst, sizes)))      # (destinations at odd places)
    launch(lib.gdn_pad_rows, dev, ctypes.addressof(segs), 4)
    torch.cuda.synchronize()
    for s, d, (a, b) in zip(src, dst, sizes):
        want = torch.zeros(*b, dtype=BF, device=DEV)
        r, c = min(a[0], b[0]), min(a[1], b[1])
        want[:r, :c] = s[:r, :c]
        n = b[0] * b[1]
        assert torch.equal(d[1:1 + n].view(b), want) and (d[:1] == 7).all() and (d[1 + n:] == 7).all()


def test_the_resizing_entry_point_refuses():
    from fla_hip import _lib
    try:
        lib = _lib.load()
    except _lib.GDNLibraryError:
        pytest.skip('not built in this checkout')
    assert lib.gdn_pad_rows(None, 1, None) == lib.gdn_pad_rows(1 << 20, 0, None) == lib.gdn_pad_rows(1 << 20, 5, None) == _lib.GDN_ERR_INVALID


@gpu
@pytest.mark.parametrize('rows', [1, 2, 4, 5, 16, 17, 300])
@pytest.mark.parametrize(('which', 'dtype'), [(w, HF) for w in ('x', 'wg', 'wu', 'wd', 'all weights')] + [(w, BF) for w in ('x', 'wg', 'wu')])
def test_operands_below_the_smallest_normal_number(rows, which, dtype):
    """fp16 numbers under 2^-14 and bf16 numbers under 2^-126 count with all their bits in every form: weights like that against rows that make up for
    them, and rows like that."""
    D, F = 264, 520
    low, high = (2.0 ** -15, 2.0 ** 12) if dtype == HF else (2.0 ** -127, 2.0 ** 120)
    t = _inputs(rows, D, F, dtype)
    for k in (('wg', 'wu', 'wd') if which == 'all weights' else (which,)):
        t[k] = (t[k].double() / t[k].double().abs().max() * low).to(dtype)
        assert (t[k] != 0).sum() > 0.9 * t[k].numel()
    if which in ('wg', 'wu', 'all weights'):
        t['x'] = (t['x'].float() * high).to(dtype)
    if which == 'x':
        t['wg'], t['wu'] = ((t[k].float() * high).to(dtype) for k in ('wg', 'wu'))
    ref = _reference(t, 'swish')['y']
    tol = _u(dtype) * ref[0].abs() + (1 + _u(dtype)) * ref[1] + TINY
    if which != 'all weights':
        assert (ref[0].abs() > tol).double().mean() > 0.5                        # (operands taken as zeros would be seen)
    with torch.no_grad():
        y = _mods().gated_mlp(t['x'], t['wg'], t['wu'], t['wd'])
    assert y.any()
    worst = ((y.double() - ref[0]).abs() / tol).max().item()
    assert worst <= 1, worst


@gpu
@pytest.mark.parametrize('rows', [1, 3, 16])
@pytest.mark.parametrize(('D', 'F'), [(1, 1), (7, 9), (31, 33), (250, 1001), (1003, 517), (2049, 40)])
def test_few_rows_of_any_width_at_any_address(rows, D, F):
    """Inference of up to 16 rows reads everything where it is."""
    t = _inputs(rows, D, F, BF)
    ref = _reference(t, 'swish')['y']

    def off(x):
        return torch.cat([x.new_full((1,), float('nan')), x.flatten(), x.new_full((9,), float('nan'))])[1:1 + x.numel()].view(x.shape)

    with torch.no_grad():
        _near('y', _mods().gated_mlp(off(t['x']), off(t['wg']), off(t['wu']), off(t['wd'])), *ref)
