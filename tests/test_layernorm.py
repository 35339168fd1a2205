"""Layer / RMS normalisation with the residual stream (fla_hip.modules: layer_norm, rms_norm, their forward and backward functions, the
layers) against the 64-bit oracle, element by element.

Tolerances, u = half the spacing of a result's type relative to it, e = 2^-24: a result is rounded once (u |ref|), and what it is formed from
is in fp32.  Statistics are sums of at most 32 terms a lane and 10 steps across lanes, so a mean is off by at most 42 e times the mean of the
magnitudes, and a few operations follow: 64 e times the magnitudes that enter covers both.  Gradients of weight and bias are sums over rows, at most
ceil(rows / 512) a lane, 16 groups and 64 steps of the last sum: 128 e times the sum of the magnitudes.  Results below the smallest normal number of fp16 are
off by half its smallest step, 2^-25."""
import contextlib
import itertools

import pytest
import torch

from oracle import modules_oracle as M

gpu = pytest.mark.gpu
DEV = 'cuda'
E = 2.0 ** -24
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _mods():
    import fla_hip.modules as mods
    return mods


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _near(name, got, ref, magnitude, steps=64):
    """|got - ref| <= u |ref| + steps e magnitude, element by element."""
    assert tuple(got.shape) == tuple(ref.shape), (name, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    tol = _u(got.dtype) * ref.abs() * (1 + 1e-3) + steps * E * magnitude + 2.0 ** -25
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1, f'{name}: {worst:.2f} of the tolerance'


def _inputs(rows, D, dtype, res, wdtype, bias, seed=0, weight=True):
    gen = torch.Generator().manual_seed(seed * 1000 + D)
    r = lambda *s: torch.randn(*s, generator=gen)
    t = dict(x=(r(rows, D) * 2 + 0.5).to(dtype).to(DEV), dy=r(rows, D).to(dtype).to(DEV))
    t['residual'] = None if res is None else (r(rows, D) * 3).to(res).to(DEV)
    t['dres'] = None if res is None else r(rows, D).to(res).to(DEV)
    t['weight'] = (1 + 0.3 * r(D)).to(wdtype).to(DEV) if weight else None
    t['bias'] = r(D).to(wdtype).to(DEV) if bias else None
    return t


def _check(t, rms, eps=1e-5, in_fp32=False, op=None, prenorm=None):
    """One forward and backward through autograd, everything against the oracle."""
    mods = _mods()
    prenorm = (t['residual'] is not None or in_fp32) if prenorm is None else prenorm
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in t.items() if k in ('x', 'residual', 'weight', 'bias') and v is not None}
    op = op or (mods.rms_norm if rms else mods.layer_norm)
    out = op(leaves['x'], leaves.get('weight'), leaves.get('bias'), residual=leaves.get('residual'), eps=eps, prenorm=prenorm, residual_in_fp32=in_fp32)
    y, stream = out if prenorm else (out, None)
    x = t['x'].double()
    exact = x if t['residual'] is None else x + t['residual'].double()
    stream_dtype = t['residual'].dtype if t['residual'] is not None else FP if in_fp32 else t['x'].dtype
    if prenorm:
        assert stream.dtype == stream_dtype
        _near('stream', stream.detach(), exact, exact.abs(), 2)
    r = stream.detach().double() if prenorm else exact.to(stream_dtype).double()       # (what the operator normalised)
    w, b = t['weight'], t['bias']
    ref, xh, rstd = M.layer_norm(r, w, b, eps, rms)
    wa = torch.ones_like(xh) if w is None else w.double().abs().expand_as(xh)
    mean = torch.zeros_like(rstd) if rms else r.abs().mean(-1, keepdim=True)
    unit = (r.abs() + mean) * rstd                                                    # (what cancels in r - mean)
    assert y.dtype == t['x'].dtype
    _near('y', y.detach(), ref, unit * wa + (0 if b is None else b.double().abs()))
    dstream = None
    if prenorm:
        dstream = t['dres'] if t['dres'] is not None else torch.randn(r.shape, generator=torch.Generator().manual_seed(3)).to(stream_dtype).to(DEV)
    names = list(leaves)
    grads = dict(zip(names, torch.autograd.grad([y] + ([stream] if prenorm else []), [leaves[k] for k in names], [t['dy']] + ([dstream] if prenorm else []))))
    dr, dw, db = M.layer_norm_grads(r, w, t['dy'], dstream, eps, rms)
    dy = t['dy'].double().abs()
    g = dy * wa
    size = rstd * (g + g.mean(-1, keepdim=True) + unit * (g * unit).mean(-1, keepdim=True)) * 2 + (0 if dstream is None else dstream.double().abs())
    for name in names:
        got = grads[name]
        assert got.dtype == leaves[name].dtype, name
        if name in ('x', 'residual'):
            _near('d' + name, got, dr, size)
        else:
            _near('d' + name, got, dw if name == 'weight' else db, (dy * unit).sum(0) if name == 'weight' else dy.sum(0), 128)
    return y.detach(), grads


FORMS = [(BF, BF, BF), (BF, FP, FP), (HF, None, FP), (FP, FP, FP), (BF, None, BF), (HF, HF, HF), (HF, FP, HF)]
# one and few features; every form of a row (16 ... 1024 lanes) on both sides of its border, aligned or not
WIDTHS = [1, 2, 7, 8, 64, 100, 128, 129, 136, 512, 520, 1000, 1001, 1024, 1032, 2048, 2050, 3000, 4096, 4100, 4104, 8192, 8200, 8203, 16000]


@gpu
@pytest.mark.parametrize(('D', 'form', 'rms', 'bias'), [(D, FORMS[i % len(FORMS)], (i // 2) % 2 == 0, i % 3 == 0) for i, D in enumerate(w for w in WIDTHS for _ in range(3))])
def test_against_the_oracle(D, form, rms, bias):
    dtype, res, wdtype = form
    _check(_inputs(37, D, dtype, res, wdtype, bias), rms)


# rows of 769 to 1024 pieces of 16 bytes that begin anywhere: 512 lanes of two
@gpu
@pytest.mark.parametrize('bias', [False, True])
@pytest.mark.parametrize('rms', [False, True])
@pytest.mark.parametrize(('dtype', 'res', 'D'), [(t, r, D) for t, widths in ((BF, (6145, 6151, 7837, 8191)), (HF, (6145, 7001, 8191)), (FP, (3073, 3077, 4095))) for D in widths
                                                 for r in {t, FP, None}])
def test_rows_of_512_lanes_at_any_address(dtype, res, D, rms, bias):
    _check(_inputs(21, D, dtype, res, FP if bias else dtype, bias), rms)


@gpu
@pytest.mark.parametrize(('dtype', 'D'), [(BF, 6152), (BF, 8192), (FP, 3076), (FP, 4096)])
def test_rows_of_512_lanes_between_16_byte_boundaries(dtype, D):
    t = _inputs(13, D, dtype, dtype, dtype, True)
    for k in ('x', 'residual', 'weight', 'bias', 'dy', 'dres'):
        t[k] = torch.cat([t[k].new_zeros(1), t[k].flatten()])[1:].view(t[k].shape)
    lib, dev = _lib_and_device()
    y, s, dx = (torch.empty_like(t['x']) for _ in range(3))
    mean, rstd = torch.empty(13, device=DEV), torch.empty(13, device=DEV)
    parts = lib.gdn_layer_norm_bwd_parts(13, D, _code(dtype))
    part = torch.empty(parts, 2, D, device=DEV)
    c = _code(dtype)
    ptr = lambda x: x.data_ptr()
    from fla_hip.ops.gated_delta_rule._common import launch
    launch(lib.gdn_layer_norm_fwd, dev, *map(ptr, (t['x'], t['residual'], t['weight'], t['bias'], y, s, mean, rstd)), 13, D, 1e-5, c, c, c, 0)
    launch(lib.gdn_layer_norm_bwd, dev, *map(ptr, (t['dy'], s, t['weight'], mean, rstd, t['dres'], dx)), None, ptr(part), 13, D, parts, 1, 1, c, c, c, 0)
    r, w, b = s.double(), t['weight'].double(), t['bias'].double()
    ref, _, rs = M.layer_norm(r, w, b, 1e-5)
    unit = (r.abs() + r.abs().mean(-1, keepdim=True)) * rs
    _near('stream', s, t['x'].double() + t['residual'].double(), (t['x'].double() + t['residual'].double()).abs(), 2)
    _near('y', y, ref, unit * w.abs() + b.abs())
    dr, dw, db = M.layer_norm_grads(r, w, t['dy'], t['dres'], 1e-5)
    dy = t['dy'].double().abs()
    g = dy * w.abs()
    _near('dx', dx, dr, rs * (g + g.mean(-1, keepdim=True) + unit * (g * unit).mean(-1, keepdim=True)) * 2 + t['dres'].double().abs())
    sums = part.double().sum(0).float()
    _near('dweight', sums[0], dw, (dy * unit).sum(0), 128)
    _near('dbias', sums[1], db, dy.sum(0), 128)


def _lib_and_device():
    from fla_hip import _lib
    return _lib.load(), torch.device('cuda', torch.cuda.current_device())


def _code(dtype):
    from fla_hip.ops.gated_delta_rule._common import dtype_code
    return dtype_code(dtype)


@gpu
@pytest.mark.parametrize('rows', [1, 3, 4, 15, 16, 17, 63, 512, 513, 1030, 4099])
@pytest.mark.parametrize('D', [64, 200, 1024, 2048])
def test_row_counts(rows, D):
    _check(_inputs(rows, D, BF, BF, BF, False), True)
    _check(_inputs(rows, D, BF, FP, FP, True), False)


@gpu
@pytest.mark.parametrize(('dtype', 'D'), [(BF, 32767), (HF, 32760), (FP, 16383), (FP, 16380), (BF, 16392)])
def test_longest_rows(dtype, D):
    _check(_inputs(19, D, dtype, dtype, FP, True), False)
    _check(_inputs(19, D, dtype, FP, FP, False), True)


@gpu
def test_without_weight_with_bias_only_and_the_stream_in_fp32():
    t = _inputs(33, 256, BF, None, BF, False, weight=False)
    _check(t, True)
    _check(t, False, in_fp32=True)
    _check(_inputs(33, 256, BF, None, BF, True, weight=False), False)
    _check(_inputs(33, 250, HF, None, HF, True), True, in_fp32=True)
    _check(_inputs(33, 256, BF, BF, BF, True), True, prenorm=False)
    _check(_inputs(33, 256, BF, None, BF, True), True, prenorm=True)              # (the stream is x itself)
    t = _inputs(33, 256, BF, BF, BF, True)
    t['bias'] = t['bias'].float()                                                 # weight and bias of two types
    _check(t, False)


@gpu
def test_values_far_from_zero_and_small_ones():
    """Rows with a mean a thousand times their spread (layer norm: two passes over registers), tiny rows under eps, large rows."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(40, 1000, generator=gen)
    for scale, shift in ((1.0, 1000.0), (1e-12, 0.0), (1e15, 0.0), (1e-3, 5.0)):
        t = _inputs(40, 1000, FP, None, FP, True)
        t['x'] = (x * scale + shift).to(DEV)
        _check(t, False)
        _check(t, True)


@gpu
@pytest.mark.parametrize('D', [64, 1000, 2048, 4096, 5000])
def test_a_row_that_is_not_finite_stays_alone(D):
    mods = _mods()
    t = _inputs(41, D, BF, BF, BF, False)
    y0, s0 = mods.rms_norm(t['x'], t['weight'], None, residual=t['residual'], prenorm=True)
    x = t['x'].clone()
    x[7, D // 2] = float('nan'); x[20] = float('inf'); x[33, 0] = -float('inf')
    y, s = mods.rms_norm(x, t['weight'], None, residual=t['residual'], prenorm=True)
    keep = torch.ones(41, dtype=torch.bool); keep[[7, 20, 33]] = False
    assert torch.equal(y[keep], y0[keep]) and torch.equal(s[keep], s0[keep])
    assert y[7].isnan().all() and y[33, 0].isnan()


@gpu
def test_strides_shapes_and_orders():
    """Transposed, sliced, expanded and misaligned tensors; any number of leading dimensions; expanded gradients."""
    mods = _mods()
    t = _inputs(24, 512, BF, BF, BF, False)
    ref = mods.rms_norm(t['x'], t['weight'], None, residual=t['residual'], prenorm=True)
    wide = torch.zeros(24, 520, dtype=BF, device=DEV); wide[:, 3:515] = t['x']
    other = torch.zeros(512, 24, dtype=BF, device=DEV).t(); other.copy_(t['residual'])
    off = torch.zeros(24 * 512 + 1, dtype=BF, device=DEV)[1:].view(24, 512); off.copy_(t['x'])
    for x in (wide[:, 3:515], off, t['x'].view(2, 3, 4, 512)):
        for res in (t['residual'], other):
            y, s = mods.rms_norm(x, t['weight'], None, residual=res.reshape(x.shape) if x.dim() > 2 else res, prenorm=True)
            assert y.shape == x.shape
            _near('y', y.reshape(24, 512), ref[0].double(), ref[0].double().abs(), 2 ** 16)        # (another form of the row: half a step of bf16)
            assert torch.equal(s.reshape(24, 512), ref[1])
    x = t['x'].clone().requires_grad_(True)
    w = t['weight'].clone().requires_grad_(True)
    (a,) = torch.autograd.grad(mods.rms_norm(x, w, None).sum(), [w])                              # an expanded gradient
    (b,) = torch.autograd.grad(mods.rms_norm(x, w, None), [w], torch.ones(24, 512, dtype=BF, device=DEV))
    assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize('D', [64, 512, 2048])
def test_fp32_tensors_on_every_16_byte_boundary(D):
    """16-bit rows with the stream, its gradient, weight and bias in fp32, each four elements off a boundary of 32 bytes."""
    t = _inputs(21, D, BF, FP, FP, True)
    for name in ('residual', 'dres', 'weight', 'bias'):
        v = t[name]
        t[name] = torch.cat([v.new_zeros(4), v.flatten()])[4:].view(v.shape)
        assert t[name].data_ptr() % 32 == 16
    mods = _mods()
    keep = {k: v.requires_grad_(True) for k, v in t.items() if k in ('x', 'residual', 'weight', 'bias')}
    y, stream = mods.layer_norm(*(keep[k] for k in ('x', 'weight', 'bias')), residual=keep['residual'], prenorm=True)
    grads = torch.autograd.grad([y, stream], list(keep.values()), [t['dy'], t['dres']])
    want = {k: v.detach().clone().requires_grad_(True) for k, v in keep.items()}
    y1, stream1 = mods.layer_norm(*(want[k] for k in ('x', 'weight', 'bias')), residual=want['residual'], prenorm=True)
    assert torch.equal(y, y1) and torch.equal(stream, stream1)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad([y1, stream1], list(want.values()), [t['dy'], t['dres'].clone()])))
    _check(_inputs(21, D, BF, FP, FP, True), False)


@gpu
def test_gradients_that_are_asked_for():
    mods = _mods()
    t = _inputs(50, 384, BF, FP, FP, True)
    args = {k: t[k].clone().requires_grad_(True) for k in ('x', 'weight', 'bias', 'residual')}
    out = mods.layer_norm(args['x'], args['weight'], args['bias'], residual=args['residual'], prenorm=True)
    full = torch.autograd.grad(out, list(args.values()), [t['dy'], t['dres']], retain_graph=True)
    for n in range(1, 4):
        for some in itertools.combinations(range(4), n):
            got = torch.autograd.grad(out, [list(args.values())[i] for i in some], [t['dy'], t['dres']], retain_graph=True)
            assert all(torch.equal(g, full[i]) for g, i in zip(got, some)), some
    # only one of the two outputs has a gradient
    a = torch.autograd.grad(out[0], args['x'], t['dy'], retain_graph=True)[0]
    b = torch.autograd.grad(out[1], args['x'], t['dres'], retain_graph=True)[0]
    _near('sum', full[0], a.double() + b.double(), a.double().abs() + b.double().abs(), 2 ** 17)    # (three roundings to bf16)
    # inputs that need none
    y = mods.layer_norm(t['x'], args['weight'], t['bias'])
    assert torch.autograd.grad(y, args['weight'], t['dy'])[0].shape == (384,)
    with torch.no_grad():
        assert not mods.layer_norm(args['x'], args['weight'], t['bias']).requires_grad


@gpu
@pytest.mark.parametrize('strided', [False, True])
@pytest.mark.parametrize('rms', [False, True])
@pytest.mark.parametrize('form', [(BF, BF, BF), (BF, FP, FP), (HF, None, FP), (BF, None, BF)])
def test_saved_tensors_may_come_back_in_another_layout_type_and_place(form, rms, strided):
    """Saved-tensor hooks on the native and on the other host path: every tensor goes to the host and comes back strided, in fp32 where it was of 16 bits, and an
    fp32 weight (of values that bf16 holds) in bf16.  What they hold is the same: so are the gradients' bits."""
    dtype, res, wdtype = form
    mods = _mods()
    t = _inputs(37, 520, dtype, res, wdtype, False)
    t['weight'] = t['weight'].to(BF).to(wdtype)
    x = t['x']
    if strided:
        x = torch.zeros(37, 528, dtype=dtype, device=DEV)[:, :520].copy_(x)

    def unpack(x):
        x = x.to(DEV)
        x = x.to(BF) if x.shape == (520,) and x.dtype == FP else x.float()
        return torch.stack([x, torch.zeros_like(x)], -1)[..., 0]

    def grads(*hooks):
        leaves = [v.detach().requires_grad_(True) for v in (x, t['weight'], t['residual']) if v is not None]
        with torch.autograd.graph.saved_tensors_hooks(*hooks) if hooks else contextlib.nullcontext():
            out = (mods.rms_norm if rms else mods.layer_norm)(leaves[0], leaves[1], None, residual=leaves[2] if res else None, prenorm=res is not None)
        return torch.autograd.grad(out, leaves, [t['dy'], t['dres']] if res else t['dy'])

    for i, (a, b) in enumerate(zip(grads(), grads(lambda x: x.cpu(), unpack))):
        assert a.dtype == b.dtype and torch.equal(a, b), i


@gpu
@pytest.mark.parametrize('strided', [False, True])
def test_saved_tensors_of_another_size_are_refused(strided):
    mods = _mods()
    x = torch.randn(6, 40 + 8 * strided, device=DEV)[:, :40].requires_grad_(True)
    for lost in ((6, 40), (40,), (6,)):
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x[:-1] if x.shape == lost else x):
            y = mods.layer_norm(x, torch.ones(40, device=DEV), None)
        with pytest.raises(ValueError, match='came back'):
            y.sum().backward()


@gpu
def test_a_second_derivative_is_refused():
    mods = _mods()
    for D in (256, 250):                                                         # (native host path; misaligned rows take the other one)
        x = torch.randn(4, D + D % 4, device=DEV)[:, :D].requires_grad_(True)
        w = torch.ones(D, device=DEV, requires_grad=True)
        (g,) = torch.autograd.grad(mods.rms_norm(x, w, None).sum(), w, create_graph=True)
        with pytest.raises(RuntimeError, match='differentiate twice'):
            g.sum().backward()


@gpu
def test_the_gradient_is_the_difference():
    """fp32: the forward kernel's own differences along a direction.  Step h = 2^-6: the third derivative leaves h^2 of order 1, rounding e / h, both below
    2e-3 of the sum of 64 x 96 terms' scale; the tolerance is 1 % of the gradient's norm along a random direction."""
    mods = _mods()
    t = _inputs(64, 96, FP, None, FP, True)
    for op in (mods.rms_norm, mods.layer_norm):
        x = t['x'].clone().requires_grad_(True)
        (g,) = torch.autograd.grad(op(x, t['weight'], t['bias']), x, t['dy'])
        v = g / g.norm() * 96 ** 0.5
        h = 2.0 ** -6
        f = lambda x: (op(x, t['weight'], t['bias']).double() * t['dy'].double()).sum()
        want = (f(t['x'] + h * v) - f(t['x'] - h * v)) / (2 * h)
        got = (g.double() * v.double()).sum()
        assert (got - want).abs() <= 0.01 * got.abs(), (got, want)


@gpu
def test_the_same_call_gives_the_same_bits_and_streams_do_not_matter():
    t = _inputs(3000, 1000, BF, BF, BF, True)
    y0, g0 = _check(t, False)
    y1, g1 = _check(t, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, g2 = _check(t, False)
    torch.cuda.current_stream().wait_stream(side)
    for y, g in ((y1, g1), (y2, g2)):
        assert torch.equal(y, y0) and all(torch.equal(g[k], g0[k]) for k in g0)


@gpu
def test_captured_and_replayed():
    """A forward and backward step in a graph: replays with new inputs, eager work between them."""
    mods = _mods()
    t = _inputs(300, 768, BF, BF, BF, False)

    def step(t):
        x, w, r = (t[k].detach().requires_grad_(True) for k in ('x', 'weight', 'residual'))
        out = mods.rms_norm(x, w, None, residual=r, prenorm=True)
        return (*(o.detach() for o in out), *torch.autograd.grad(out, [x, w, r], [t['dy'], t['dres']]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(t)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(t)
    for seed in range(4):
        new = _inputs(300, 768, BF, BF, BF, False, seed=seed + 5)
        eager = step(new)
        for k, v in new.items():
            if v is not None:
                t[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b), seed


@gpu
def test_more_elements_than_32_bits_count():
    mods = _mods()
    rows, D = 1_100_003, 2048
    x = torch.zeros(rows, D, dtype=BF, device=DEV)
    tail = _inputs(5, D, BF, None, BF, False)
    x[-5:] = tail['x']
    x.requires_grad_(True)
    w = tail['weight'].clone().requires_grad_(True)
    y = mods.rms_norm(x, w, None)
    ref = mods.rms_norm(tail['x'], w, None)
    assert torch.equal(y[-5:], ref) and not y[:-5].any()
    dy = torch.zeros_like(y)
    dy[-5:] = tail['dy']
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    xt = tail['x'].clone().requires_grad_(True)
    rx, rw = torch.autograd.grad(mods.rms_norm(xt, w, None), [xt, w], tail['dy'])
    assert torch.equal(dx[-5:], rx) and not dx[:-5].any()
    _near('dw', dw, rw.double(), rw.double().abs(), 2 ** 17)


@gpu
def test_no_rows():
    mods = _mods()
    w = torch.ones(96, device=DEV, requires_grad=True)
    x = torch.zeros(0, 96, device=DEV, requires_grad=True)
    y, s = mods.rms_norm(x, w, None, residual=torch.zeros(0, 96, device=DEV), prenorm=True)
    assert y.shape == s.shape == (0, 96)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert dx.shape == (0, 96) and not dw.any()
    assert mods.layer_norm(torch.zeros(3, 0, 96, device=DEV), w, None).shape == (3, 0, 96)


@gpu
def test_the_entry_points_write_their_rows_only():
    """Through the C ABI into the middle of larger buffers: what lies around stays."""
    from fla_hip import _lib
    from fla_hip.ops.gated_delta_rule._common import launch, ptr
    for rows, D in ((13, 100), (13, 1001), (5, 2048), (3, 5000)):
        t = _inputs(rows, D, BF, BF, BF, False)
        big = torch.full((4, rows * D + 64), 7.0, dtype=BF, device=DEV)
        y, s, dx = (big[i, 32:32 + rows * D] for i in range(3))
        rstd = torch.empty(rows, device=DEV)
        lib, dev = _lib.load(), torch.device('cuda', torch.cuda.current_device())
        launch(lib.gdn_layer_norm_fwd, dev, ptr(t['x']), ptr(t['residual']), ptr(t['weight']), None, ptr(y), ptr(s), None, ptr(rstd), rows, D, 1e-5, 0, 0, 0, 1)
        parts = lib.gdn_layer_norm_bwd_parts(rows, D, 0)
        part = torch.full((parts * D + 64,), 7.0, device=DEV)
        launch(lib.gdn_layer_norm_bwd, dev, ptr(t['dy']), ptr(s), ptr(t['weight']), None, ptr(rstd), None, ptr(dx), None, ptr(part), rows, D, parts, 1, 0, 0, 0, 0, 1)
        torch.cuda.synchronize()
        ref = M.layer_norm(s.view(rows, D), t['weight'], None, 1e-5, True)[0]
        _near('y', y.view(rows, D), ref, ref.abs())
        assert (big[:, :32] == 7).all() and (big[:, 32 + rows * D:] == 7).all() and (big[3] == 7).all() and (part[parts * D:] == 7).all()


@gpu
def test_the_layers():
    mods = _mods()
    ln = mods.LayerNorm(384, bias=True, device=DEV, dtype=BF)
    rms = mods.RMSNorm(384, eps=1e-6, device=DEV, dtype=BF)
    plain = mods.RMSNorm(384, elementwise_affine=False, device=DEV)
    assert {n for n, _ in ln.named_parameters()} == {'weight', 'bias'} and {n for n, _ in rms.named_parameters()} == {'weight'}
    assert repr(rms) == 'RMSNorm(384, eps=1e-06)' and list(plain.parameters()) == []
    x = torch.randn(2, 9, 384, device=DEV).to(BF)
    with torch.no_grad():
        ln.weight.normal_(1, 0.2); ln.bias.normal_(); rms.weight.normal_(1, 0.2)
    r = x.double()
    for m, ref in ((ln, M.layer_norm(r, ln.weight, ln.bias, 1e-5)[0]), (rms, M.layer_norm(r, rms.weight, None, 1e-6, True)[0]), (plain, M.layer_norm(r, None, None, 1e-5, True)[0])):
        _near(repr(m), m(x).detach(), ref, ref.abs() + 2)
    y, s = rms(x, residual=x, prenorm=True, residual_in_fp32=True)
    assert s.dtype == BF and torch.equal(s, x + x)
    rms(x).sum().backward()
    assert rms.weight.grad.shape == (384,)


def _refusals():
    z = torch.zeros
    half = z(4, 8, dtype=HF)
    return [
        ('a weight of another width', ValueError, lambda m: m.layer_norm_fwd(z(4, 8), z(7), None)),
        ('rows without features', ValueError, lambda m: m.layer_norm_fwd(z(4, 0), None, None)),
        ('three dimensions', ValueError, lambda m: m.layer_norm_fwd(z(4, 8, 2), None, None)),
        ('a residual of another shape', ValueError, lambda m: m.rms_norm(z(4, 8), None, None, residual=z(4, 9))),
        ('a residual of another 16-bit type', NotImplementedError, lambda m: m.rms_norm(half, None, None, residual=half.bfloat16())),
        ('a residual narrower than x', NotImplementedError, lambda m: m.rms_norm(z(4, 8), None, None, residual=half)),
        ('64 bits', NotImplementedError, lambda m: m.rms_norm(z(4, 8, dtype=torch.float64), None, None)),
        ('rows of 64 KB', RuntimeError, lambda m: m.rms_norm(z(1, 32768, dtype=BF), None, None)),
        ('no dimension', ValueError, lambda m: m.rms_norm(z(()), None, None)),
        ('a backward without statistics', ValueError, lambda m: m.layer_norm_bwd(z(4, 8), z(4, 8), z(8), None)),
        ('layer norm without means', ValueError, lambda m: m.layer_norm_bwd(z(4, 8), z(4, 8), z(8), None, rstd=z(4))),
        ('a gradient of another shape', ValueError, lambda m: m.layer_norm_bwd(z(4, 9), z(4, 8), z(8), None, rstd=z(4), is_rms_norm=True)),
        ('statistics of another length', ValueError, lambda m: m.layer_norm_bwd(z(4, 8), z(4, 8), z(8), None, rstd=z(5), is_rms_norm=True)),
    ]


@pytest.mark.parametrize(('what', 'error', 'call'), _refusals(), ids=[r[0] for r in _refusals()])
def test_refusals(what, error, call, monkeypatch):
    from fla_hip.modules import layernorm
    monkeypatch.setattr(layernorm, 'require_gpu', lambda x, *_: x.device)         # (what is wrong is found before anything else is asked)
    with pytest.raises(error):
        call(layernorm)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match='GPU'):
        _mods().rms_norm(torch.zeros(4, 8), None, None)


def test_the_entry_points_refuse():
    """By the library's host code: nothing is launched."""
    from fla_hip import _lib
    try:
        lib = _lib.load()
    except _lib.GDNLibraryError:
        pytest.skip('not built in this checkout')
    P = 1 << 20                                                                    # (an address that is never read)
    fwd = lambda rows=4, D=8, x=P, y=P, res=None, out=None, dt=0, sdt=0, wdt=0: lib.gdn_layer_norm_fwd(x, res, P, None, y, out, None, None, rows, D, 1e-5, dt, sdt, wdt, 1, None)
    assert fwd(rows=-1) == fwd(D=0) == fwd(x=None) == fwd(y=None) == fwd(res=P) == _lib.GDN_ERR_INVALID
    assert fwd(D=32769) == fwd(D=16385, dt=2, sdt=2) == fwd(sdt=1) == fwd(dt=2, sdt=0) == fwd(dt=9) == fwd(wdt=1) == _lib.GDN_ERR_UNSUPPORTED
    assert fwd(rows=0) == _lib.GDN_OK
    bwd = lambda rows=4, D=8, dy=P, rstd=P, mean=None, part=P, parts=1, dw=1, rms=1, dt=0: lib.gdn_layer_norm_bwd(
        dy, P, P, mean, rstd, None, P, None, part, rows, D, parts, dw, 0, dt, dt, dt, rms, None)
    assert bwd(parts=0) == bwd(parts=65536) == bwd(part=None) == bwd(dy=None) == bwd(rstd=None) == bwd(rms=0) == _lib.GDN_ERR_INVALID
    assert bwd(D=32769) == _lib.GDN_ERR_UNSUPPORTED
    assert bwd(rows=0, dw=0) == _lib.GDN_OK
