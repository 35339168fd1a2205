"""The steps of a Gated DeltaNet block around the token mixing - normalisation with the residual stream, gated feed-forward block - as
cases that can be prepared, run and compared.

Four kinds of work:
  norm         layer norm or RMS norm of rows, the residual stream added first and handed on (prenorm): ``layer_norm``, ``rms_norm``
  norm_train   the same with the gradients of x, the residual stream, weight and bias
  mlp          y = (act(x Wg^T) * (x Wu^T)) Wd^T: ``gated_mlp``
  mlp_train    the same with the gradients of x and the three weights

``own`` false: the plain form, elementary torch operations in 32 bits rounded once at the end.  ``own`` true: the framework's calls.
``exact`` gives the same results from the definitions in 64 bits."""
import importlib
import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
BYTES = {'bf16': 2, 'f16': 2, 'f32': 4}
MOST_MLP = 3 * 8192 * 4096 * 11008      # tokens x hidden x intermediate of the largest training step (three forwards' work)
MOST_NORM = 16384 * 4096                # elements of the largest training step of the norm


def listed():
    return [
        # One user's next token: the norm in front of the feed-forward block on a single row.  Launch and host time.
        dict(name='norm_step', kind='norm', rms=True, rows=1, D=2048, dtype='bf16', wdtype='bf16', residual='bf16', bias=False),
        # A long document's prefill at the layer's default width, the residual stream added and handed on.
        dict(name='norm_prefill', kind='norm', rms=True, rows=32768, D=2048, dtype='bf16', wdtype='bf16', residual='bf16', bias=False),
        # A training step of a wide model, the residual stream kept in 32 bits.
        dict(name='norm_train', kind='norm_train', rms=True, rows=16384, D=4096, dtype='bf16', wdtype='f32', residual='f32', bias=False),
        # Layer norm with bias on rows of no round length, no residual stream: a packed batch's leftover of a small model.
        dict(name='norm_train_odd', kind='norm_train', rms=False, rows=4099, D=1001, dtype='f16', wdtype='f16', residual='none', bias=True),
        # One token through the feed-forward block: every weight is read once.
        dict(name='mlp_step_1', kind='mlp', tokens=1, D=2048, F=5632, dtype='bf16', act='swish'),
        # A decode step of a small batch.
        dict(name='mlp_step_48', kind='mlp', tokens=48, D=2048, F=5632, dtype='bf16', act='swish'),
        # A short question, of no round length.
        dict(name='mlp_prefill_short', kind='mlp', tokens=333, D=2048, F=5632, dtype='f16', act='swish'),
        # A long document.
        dict(name='mlp_prefill_long', kind='mlp', tokens=32768, D=2048, F=5632, dtype='bf16', act='swish'),
        # A training step at the layer's default width ...
        dict(name='mlp_train', kind='mlp_train', tokens=8192, D=2048, F=5632, dtype='bf16', act='swish'),
        # ... of a small odd model on a ragged batch ...
        dict(name='mlp_train_odd', kind='mlp_train', tokens=2999, D=1004, F=2690, dtype='f16', act='gelu_tanh'),
        # ... and of a wide one.
        dict(name='mlp_train_wide', kind='mlp_train', tokens=8192, D=4096, F=11008, dtype='bf16', act='swish'),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(['norm', 'norm_train', 'mlp', 'mlp_train'], [2, 3, 4, 4])[0]
    if kind.startswith('norm'):
        dtype = rng.choices(['bf16', 'f16', 'f32'], [4, 1, 1])[0]
        D = rng.choice([rng.choice([1024, 2048, 4096]), 8 * _log_int(rng, 8, 1024), _log_int(rng, 60, 8192)])
        rows = _log_int(rng, 1 if kind == 'norm' else 64, min(32768, MOST_NORM // D))
        rms = rng.random() < 0.7
        return dict(kind=kind, rms=rms, rows=rows, D=D, dtype=dtype, wdtype=rng.choice([dtype, 'f32']),
                    residual=rng.choice(['none', dtype, 'f32']), bias=not rms and rng.random() < 0.7)
    D = rng.choice([rng.choice([1024, 2048, 4096]), 8 * _log_int(rng, 32, 512), _log_int(rng, 250, 4096)])
    F = rng.choice([256 * -(-8 * D // 768), 8 * _log_int(rng, D // 8, D // 2), _log_int(rng, D, 4 * D)])
    train = kind == 'mlp_train'
    tokens = _log_int(rng, 16 if train else 1, min(32768, MOST_MLP // (D * F) // (3 if train else 1)))
    return dict(kind=kind, tokens=tokens, D=D, F=F, dtype=rng.choices(['bf16', 'f16'], [3, 1])[0], act=rng.choices(['swish', 'gelu_tanh', 'sigmoid'], [4, 1, 1])[0])


def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device='cuda') * std).to(DTYPES[dtype])


def _inputs(case, seed):
    """Rows as a trained network's stream has them (unit values, one feature in 64 eight times as large), weights of the usual scale."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    D, dt = case['D'], case['dtype']
    loud = torch.where(torch.arange(D, device='cuda') % 64 == 5, 8.0, 1.0)
    if case['kind'].startswith('norm'):
        n, res = case['rows'], case['residual']
        t = dict(x=(torch.randn(n, D, generator=gen, device='cuda') * loud).to(DTYPES[dt]),
                 weight=(1 + 0.2 * torch.randn(D, generator=gen, device='cuda')).to(DTYPES[case['wdtype']]))
        if case['bias']:
            t['bias'] = _normal(gen, (D,), case['wdtype'], 0.1)
        if res != 'none':
            t['residual'] = _normal(gen, (n, D), res, 2.0)
        if case['kind'] == 'norm_train':
            t['dy'] = _normal(gen, (n, D), dt)
            if res != 'none':
                t['dres'] = _normal(gen, (n, D), res)
        return t
    n, F = case['tokens'], case['F']
    t = dict(x=_normal(gen, (n, D), dt), wg=_normal(gen, (F, D), dt, D ** -0.5), wu=_normal(gen, (F, D), dt, D ** -0.5), wd=_normal(gen, (D, F), dt, F ** -0.5))
    if case['kind'] == 'mlp_train':
        t['dy'] = _normal(gen, (n, D), dt)
    return t


LEAVES = ('x', 'residual', 'weight', 'bias', 'wg', 'wu', 'wd')


def prepare(case, seed):
    t = _inputs(case, seed)
    if case['kind'].endswith('_train'):
        for name in LEAVES:
            if name in t:
                t[name].requires_grad_(True)
    return dict(case=case, eps=1e-6, **t)


_modules = None


def _framework():
    global _modules
    if _modules is None:
        importlib.import_module('flash-linear-attention_amd')
        import fla_hip.modules as _modules
    return _modules


def run(s):
    train = s['case']['kind'].endswith('_train')
    if own:
        # (inference runs without a graph, as a serving program does)
        with torch.set_grad_enabled(train):
            return _run_own(s, train)
    with torch.no_grad():
        return _plain_norm(s) if 'weight' in s else _plain_mlp(s)


def _run_own(s, train):
    modules, case = _framework(), s['case']
    if 'weight' in s:
        op = modules.rms_norm if case['rms'] else modules.layer_norm
        res = s.get('residual')
        out = op(s['x'], s['weight'], s.get('bias'), residual=res, eps=s['eps'], prenorm=res is not None)
        outs = dict(zip(('y', 'stream'), out)) if res is not None else dict(y=out)
        douts = [s[k] for k in ('dy', 'dres') if k in s]
    else:
        outs = dict(y=modules.gated_mlp(s['x'], s['wg'], s['wu'], s['wd'], activation=case['act']))
        douts = [s.get('dy')]
    if not train:
        return outs
    names = [n for n in LEAVES if n in s]
    grads = torch.autograd.grad(list(outs.values()), [s[n] for n in names], douts)
    return {**{k: v.detach() for k, v in outs.items()}, **{'d' + n: g for n, g in zip(names, grads)}}


def _plain_norm(s):
    case, x, w = s['case'], s['x'], s['weight'].float()
    r = x.float()
    res = s.get('residual')
    if res is not None:
        # what is normalised is the stream as it is handed on, in its own type
        stream = (r + res.float()).to(res.dtype)
        r = stream.float()
    rc = r if case['rms'] else r - r.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((rc * rc).mean(-1, keepdim=True) + s['eps'])
    xh = rc * rstd
    y = xh * w
    if case['bias']:
        y = y + s['bias'].float()
    out = dict(y=y.to(x.dtype))
    if res is not None:
        out['stream'] = stream
    if case['kind'] == 'norm_train':
        dy = s['dy'].float()
        dxh = dy * w
        dr = dxh - xh * (dxh * xh).mean(-1, keepdim=True)
        if not case['rms']:
            dr = dr - dxh.mean(-1, keepdim=True)
        dr = dr * rstd
        if res is not None:
            dr = dr + s['dres'].float()
            out['dresidual'] = dr.to(res.dtype)
        out['dx'] = dr.to(x.dtype)
        out['dweight'] = (dy * xh).sum(0).to(s['weight'].dtype)
        if case['bias']:
            out['dbias'] = dy.sum(0).to(s['bias'].dtype)
    return out


_GELU = math.sqrt(2 / math.pi)


def _act(kind, g):
    """The activation and its derivative."""
    if kind == 'gelu_tanh':
        t = torch.tanh(_GELU * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * _GELU * (1 + 0.134145 * g * g)
    sig = 1 / (1 + torch.exp(-g))
    if kind == 'sigmoid':
        return sig, sig * (1 - sig)
    return g * sig, sig * (1 + g * (1 - sig))


def _plain_mlp(s):
    dt = s['x'].dtype
    x, wg, wu, wd = (s[k].float() for k in ('x', 'wg', 'wu', 'wd'))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(s['case']['act'], g)
    h = a * u
    out = dict(y=(h @ wd.t()).to(dt))
    if 'dy' in s:
        dy = s['dy'].float()
        dh = dy @ wd
        dg, du = dh * u * da, dh * a
        out['dx'] = (dg @ wg + du @ wu).to(dt)
        out['dwg'], out['dwu'], out['dwd'] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt), (dy.t() @ h).to(dt)
    return out


def exact(case, seed):
    t = {k: v.double() for k, v in _inputs(case, seed).items()}
    x = t['x']
    if case['kind'].startswith('norm'):
        w, b = t['weight'], t.get('bias', 0.0)
        # (the stream is a tensor of the residual's type, and that tensor is normalised)
        stream = (x + t['residual']).to(DTYPES[case['residual']]).double() if 'residual' in t else x
        mu = 0.0 if case['rms'] else stream.sum(1, keepdim=True) / case['D']
        var = ((stream - mu) ** 2).sum(1, keepdim=True) / case['D']
        unit = (stream - mu) * (var + 1e-6) ** -0.5
        out = dict(y=unit * w + b)
        if 'residual' in t:
            out['stream'] = stream
        if 'dy' in t:
            # d unit / d stream: the projection that takes away what lies along `unit` (and, centred, along ones), over the deviation
            du = t['dy'] * w
            along = (du * unit).sum(1, keepdim=True) / case['D'] * unit
            if not case['rms']:
                along = along + du.sum(1, keepdim=True) / case['D']
            out['dx'] = (du - along) * (var + 1e-6) ** -0.5 + t.get('dres', 0.0)
            if 'residual' in t:
                out['dresidual'] = out['dx']
            out['dweight'] = (unit * t['dy']).sum(0)
            if case['bias']:
                out['dbias'] = t['dy'].sum(0)
        return out
    g, u = torch.mm(x, t['wg'].t()), torch.mm(x, t['wu'].t())
    if case['act'] == 'gelu_tanh':
        inner = _GELU * (g + 0.044715 * g ** 3)
        a = g * torch.sigmoid(2 * inner)                            # (1 + tanh z) / 2 = sigmoid(2 z)
        da = torch.sigmoid(2 * inner) + a * torch.sigmoid(-2 * inner) * 2 * _GELU * (1 + 3 * 0.044715 * g ** 2)
    elif case['act'] == 'sigmoid':
        a = torch.sigmoid(g)
        da = a * torch.sigmoid(-g)
    else:
        a = g * torch.sigmoid(g)
        da = torch.sigmoid(g) + a * torch.sigmoid(-g)
    out = dict(y=torch.mm(a * u, t['wd'].t()))
    if 'dy' in t:
        dh = torch.mm(t['dy'], t['wd'])
        out['dwd'] = torch.mm(t['dy'].t().contiguous(), a * u)
        dg, du = dh * da * u, dh * a
        out['dx'] = torch.mm(dg, t['wg']) + torch.mm(du, t['wu'])
        out['dwg'], out['dwu'] = torch.mm(dg.t().contiguous(), x), torch.mm(du.t().contiguous(), x)
    return out


def work(case):
    D, b, train = case['D'], BYTES[case['dtype']], case['kind'].endswith('_train')
    if case['kind'].startswith('norm'):
        n, res, wb = case['rows'], BYTES.get(case['residual'], 0), BYTES[case['wdtype']] * (2 if case['bias'] else 1)
        # x and the residual in, y and the stream out; dy and the stream's gradient in, dx and the residual's gradient out; parameters
        # and their gradients
        byts = n * D * (2 * b + 2 * res) * (2 if train else 1) + D * wb * (2 if train else 1)
        return dict(bytes=byts, flops=n * D * (16 if train else 6))
    n, F = case['tokens'], case['F']
    byts = b * (2 * n * D + 3 * D * F) * (2 if train else 1)
    return dict(bytes=byts, flops=(18 if train else 6) * n * D * F)
