"""The paged cache (fla_hip.ops.attn: paged_append, paged_keep): every slot of the cache after a call against the definition, those that are not written bit for bit.

Keys that are turned on the way are off by what tests/test_rotary.py derives (three roundings of e = 2^-24 of the magnitudes that enter, and one of the result);
everything else is copied."""
import os
import subprocess

import pytest
import torch

from oracle import serving_oracle as O
from paged_inputs import DEV, cache, pages_for, table

gpu = pytest.mark.gpu
E = 2.0 ** -24
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _attn():
    from fla_hip.ops import attn
    return attn


def _near(got, ref, size):
    got = got.cpu()
    u = torch.finfo(got.dtype).eps / 2
    tol = u * ref.abs() * (1 + 1e-3) + 3 * E * size + (2.0 ** -25 if got.dtype == HF else 2.0 ** -140)
    assert ((got.double() - ref).abs() <= tol).all(), ((got.double() - ref).abs() / tol).max()


def _rows(*shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _tables(positions, R):
    t = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return t.cos().float().to(DEV), t.sin().float().to(DEV)


def _append(contexts, rows, page_size, HQ, HK, D, R, dtype, packed=False, layout='slots', index=torch.int32, positions=None, interleaved=False, spoil=None, strided=False):
    """One call against the definition.  spoil(table): changes the table before the call."""
    N = len(contexts)
    lengths = [c + r for c, r in zip(contexts, rows)]
    pages = pages_for(lengths, page_size)
    k_cache, v_cache = cache(pages, page_size, HK, D, dtype, layout=layout)
    t = table(lengths, page_size, pages)
    if spoil:
        spoil(t)
    shape = (1, sum(rows)) if packed else (N, rows[0])
    if strided:                                                  # parts of one projection's result
        qkv = _rows(*shape, (HQ + 2 * HK) * D, dtype=dtype)
        q, k, v = (x.view(*shape, -1, D) for x in qkv.split([HQ * D, HK * D, HK * D], -1))
    else:
        q, k, v = (_rows(*shape, h, D, dtype=dtype, seed=i) for i, h in enumerate((HQ, HK, HK)))
    cos, sin = _tables(max(lengths) + 4, R) if R else (None, None)
    cu = torch.tensor([0, *torch.tensor(rows).cumsum(0).tolist()], dtype=index, device=DEV) if packed else None
    firsts = [0, *torch.tensor(rows).cumsum(0).tolist()]
    at = torch.zeros(shape, dtype=torch.long)
    for n in range(N):
        at.view(-1)[firsts[n]:firsts[n + 1]] = torch.arange(rows[n]) + contexts[n]
    if positions is not None:
        turned_at = positions(at)
        given = turned_at.to(index).to(DEV)
    else:
        turned_at, given = at, None
    before = k_cache.clone(), v_cache.clone()
    out = _attn().paged_append(k, v, k_cache, v_cache, t.to(DEV), torch.tensor(contexts, dtype=index, device=DEV), cu_seqlens=cu, q=q if HQ else None, cos=cos, sin=sin,
                               positions=given, interleaved=interleaved)
    want_k, want_v, size = before[0].double().cpu(), before[1].clone().cpu(), torch.zeros(before[0].shape, dtype=torch.float64)
    if R:
        turned, k_size = O.rotary(k, cos, sin, turned_at, interleaved)
        want_q, q_size = O.rotary(q, cos, sin, turned_at, interleaved)
    else:
        turned, k_size, want_q, q_size = k.double().cpu(), torch.zeros(k.shape), q.double().cpu(), torch.zeros(q.shape)
    written = torch.zeros(pages, page_size, dtype=torch.bool)
    for n in range(N):
        for i in range(rows[n]):
            slot = O.slot_of(t, n, contexts[n] + i, pages, page_size)
            if slot is None:
                continue
            row = firsts[n] + i
            want_k[slot], size[slot], want_v[slot] = turned.flatten(0, 1)[row], k_size.flatten(0, 1)[row].double(), v.cpu().flatten(0, 1)[row]
            written[slot] = True
    _near(k_cache, want_k, size)
    assert torch.equal(k_cache.cpu()[~written], before[0].cpu()[~written]) and torch.equal(v_cache.cpu(), want_v)
    if HQ:
        assert out.is_contiguous()
        _near(out, want_q, q_size)
    else:
        assert out is None
    return written


@gpu
@pytest.mark.parametrize('packed', [False, True])
@pytest.mark.parametrize(('page_size', 'HQ', 'HK', 'D', 'R', 'dtype'), [
    (16, 4, 2, 128, 128, BF), (1, 2, 1, 64, 64, HF), (10, 6, 3, 80, 80, HF), (64, 8, 8, 256, 64, BF), (7, 0, 2, 128, 0, BF), (16, 3, 1, 72, 36, BF), (33, 5, 5, 100, 50, FP), (5, 1, 1, 33, 0, HF)])
def test_append(page_size, HQ, HK, D, R, dtype, packed):
    for contexts, rows in (([0], [1]), ([31, 0, 16], [3, 3, 3]), ([5, 64, 0, 100], [1, 40, 0, 7] if packed else [9, 9, 9, 9])):
        written = _append(contexts, rows, page_size, HQ, HK, D, R, dtype, packed)
        assert int(written.sum()) == sum(rows)


@gpu
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('layout', ['heads', 'one', 'odd'])
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
def test_append_to_other_layouts(layout, index, interleaved):
    _append([11, 3], [6, 6], 8, 4, 2, 64, 32, BF, False, layout, index, interleaved=interleaved, strided=True)


@gpu
def test_append_at_positions_of_a_tree():
    depth = torch.tensor([0, 1, 1, 2, 2, 2])
    _append([11, 3], [6, 6], 8, 4, 2, 64, 64, BF, positions=lambda at: at[:, :1] + depth)
    _append([11, 3], [6, 2], 8, 4, 2, 64, 64, BF, packed=True, positions=lambda at: at + torch.arange(8) % 2)


def _no_page(t):
    t[0, 1] = -1
    t[1, 0] = 10 ** 6
    t[2, 0] = -2 ** 31


@gpu
@pytest.mark.parametrize('page_size', [4, 16])
def test_rows_without_a_page_write_nothing(page_size):
    written = _append([2, 0, 1], [page_size, page_size, page_size], page_size, 2, 1, 64, 64, BF, spoil=_no_page)
    assert 0 < int(written.sum()) < 3 * page_size
    # the table's row ends before the slots do
    k_cache, v_cache = cache(4, 4, 1, 64, BF)
    before = k_cache.clone()
    k = _rows(1, 6, 1, 64, dtype=BF)
    _attn().paged_append(k, k, k_cache, v_cache, torch.tensor([[2]], dtype=torch.int32, device=DEV), torch.tensor([1], device=DEV))
    assert torch.equal(k_cache[2, 1:], k[0, :3]) and torch.equal(k_cache[[0, 1, 3]], before[[0, 1, 3]]) and torch.equal(k_cache[2, 0], before[2, 0])
    _attn().paged_append(k, k, k_cache, v_cache, torch.zeros(1, 0, dtype=torch.int32, device=DEV), torch.tensor([0], device=DEV))
    _attn().paged_append(k, k, k_cache, v_cache, torch.tensor([[0]], dtype=torch.int32, device=DEV), torch.tensor([-9], device=DEV))
    assert torch.equal(k_cache[0], before[0])


@gpu
def test_rows_of_no_sequence_write_nothing():
    k_cache, v_cache = cache(4, 4, 2, 64, BF)
    before = k_cache.clone()
    q, k = _rows(1, 9, 2, 64, dtype=BF), _rows(1, 9, 2, 64, dtype=BF, seed=1)
    cos, sin = _tables(16, 64)
    t = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32, device=DEV)
    for max_seqlen in (None, 9):
        out = _attn().paged_append(k, k, k_cache, v_cache, t, torch.tensor([2, 0], device=DEV), cu_seqlens=torch.tensor([1, 4, 6], device=DEV), max_seqlen=max_seqlen, q=q, cos=cos, sin=sin)
        touched = torch.zeros(4, 4, dtype=torch.bool)
        touched[3, 2:], touched[1, :1], touched[0, :2] = True, True, True
        assert torch.equal(k_cache.cpu()[~touched], before.cpu()[~touched])
        assert torch.equal(out[0, [0, 6, 7, 8]], q[0, [0, 6, 7, 8]])
        _near(out[:, 1:6], *O.rotary(q[:, 1:6], cos, sin, torch.tensor([[2, 3, 4, 0, 1]])))


@gpu
@pytest.mark.parametrize('layout', ['slots', 'heads', 'odd'])
@pytest.mark.parametrize(('page_size', 'D', 'dtype'), [(16, 128, BF), (3, 64, HF), (1, 40, BF), (64, 33, HF), (10, 256, FP)])
def test_keep(page_size, D, dtype, layout):
    paths = [[0, 2, 3, 7], [0], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10], [0, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 17], [0, 1, 5]]
    contexts, R = [0, 5, 33, 16, 7], 18
    lengths = [c + R for c in contexts]
    pages = pages_for(lengths, page_size)
    k_cache, v_cache = cache(pages, page_size, 2, D, dtype, layout=layout)
    t = table(lengths, page_size, pages)
    rows = torch.full((5, R), -1, dtype=torch.int32)
    for n, path in enumerate(paths):
        rows[n, :len(path)] = torch.tensor(path)
    kept = torch.tensor([len(p) for p in paths])
    want = [c.clone().cpu() for c in (k_cache, v_cache)]
    for n, path in enumerate(paths):
        for c, now in zip(want, (k_cache.cpu(), v_cache.cpu())):
            for i, r in enumerate(path):
                c[O.slot_of(t, n, contexts[n] + i, pages, page_size)] = now[O.slot_of(t, n, contexts[n] + r, pages, page_size)]
    _attn().paged_keep(k_cache, v_cache, t.to(DEV), torch.tensor(contexts, device=DEV), rows.to(DEV), kept.to(DEV))
    assert torch.equal(k_cache.cpu(), want[0]) and torch.equal(v_cache.cpu(), want[1])


@gpu
def test_keep_leaves_what_may_not_move():
    k_cache, v_cache = cache(6, 4, 2, 64, BF)
    t = torch.tensor([[4, 1, 3], [0, -1, 2], [5, 5000, -7]], dtype=torch.int32)
    rows = torch.tensor([[0, 0, -1, 5, 100, 2 ** 31 - 1], [1, 5, 2, 6, 4, 5], [3, 2, 6, 3, 8, 5]], dtype=torch.int32)
    kept, contexts = torch.tensor([99, 6, 5], dtype=torch.int32), torch.tensor([1, 1, 0], dtype=torch.int32)
    want = [c.clone().cpu() for c in (k_cache, v_cache)]
    for n in range(3):
        for i in range(min(int(kept[n]), 6)):
            r = int(rows[n, i])
            fro, to = (O.slot_of(t, n, int(contexts[n]) + x, 6, 4) for x in (r, i))
            if r > i and fro and to:
                for c, now in zip(want, (k_cache.cpu(), v_cache.cpu())):
                    c[to] = now[fro]
    _attn().paged_keep(k_cache, v_cache, t.to(DEV), contexts.to(DEV), rows.to(DEV), kept.to(DEV))
    assert torch.equal(k_cache.cpu(), want[0]) and torch.equal(v_cache.cpu(), want[1])
    after = k_cache.clone()
    _attn().paged_keep(k_cache, v_cache, t.to(DEV), contexts.to(DEV), rows.to(DEV), torch.tensor([-5, 0, 1], device=DEV))
    assert torch.equal(k_cache, after)                           # (the one row that may move had moved before)


@gpu
def test_written_caches_are_noticed_by_a_graph_that_saved_them():
    k_cache, v_cache = cache(2, 4, 1, 16, FP)
    x = torch.ones_like(k_cache).requires_grad_()
    k = _rows(1, 1, 1, 16, dtype=FP)
    t, context = torch.tensor([[1]], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    loss = (x * k_cache).sum()
    _attn().paged_append(k, k, k_cache, v_cache, t, context)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


_INDEX_TEST = r'''
#include "gdn_paged_index.h"
#include <cstdio>
#include <vector>
using namespace gdn;
int main() {
    // the table's rows stand in a larger array that must not be read outside of them (built with the address sanitizer)
    const int cols = 3, stride = 4;
    std::vector<int32_t> table = {0, 4, -1, 99, 5, 2147483647, -2147483647 - 1};
    const PageTable t{table.data(), stride, cols * 7, 5, 7};
    const int want[2][3] = {{0, 4, -1}, {-1, -1, -1}};
    for (int64_t slot : {(int64_t)-1, (int64_t)-9000000000, (int64_t)21, (int64_t)9000000000, INT64_MAX, INT64_MIN})
        for (int n = 0; n < 2; ++n)
            if (page_of(t, n, slot) != -1) return printf("slot %lld\n", (long long)slot), 1;
    for (int n = 0; n < 2; ++n)
        for (int slot = 0; slot < 21; ++slot)
            if (page_of(t, n, slot) != want[n][slot / 7]) return printf("slot %d of %d\n", slot, n), 1;
    const PageTable none{nullptr, 0, 0, 5, 7};
    if (page_of(none, 0, 0) != -1) return 1;
    // every row of every batch of up to four boundaries, whatever they are: the answer is right where they do not decrease, and no other boundary is read
    for (int N = 1; N <= 3; ++N)
        for (int code = 0; code < 6 * 6 * 6 * 6; ++code) {
            std::vector<int64_t> cu;
            for (int k = 0, c = code; k <= N; ++k, c /= 6) cu.push_back(c % 6 - 1);
            bool sorted = true;
            for (int k = 0; k < N; ++k) sorted = sorted && cu[k] <= cu[k + 1];
            for (int64_t row = 0; row < 5; ++row) {
                const int64_t n = sequence_of(row, N, [&](int64_t k) { return cu.at(k); });
                int64_t right = -1;
                for (int k = 0; k < N; ++k)
                    if (cu[k] <= row && row < cu[k + 1]) right = k;
                if (n < -1 || n >= N || (n >= 0 && !(cu[n] <= row && row < cu[n + 1])) || (sorted && n != right)) return printf("row %lld\n", (long long)row), 1;
            }
        }
    puts("ok");
}
'''


def test_places_in_the_cache_on_the_host(tmp_path):
    """The code that the kernels find slots and sequences with, as a program of the host: no number in a table, a length or a boundary leads outside."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, exe = tmp_path / 'index.cpp', tmp_path / 'index'
    src.write_text(_INDEX_TEST)
    subprocess.run(['g++', '-std=c++17', '-g', '-fsanitize=address,undefined', '-static-libasan', f'-I{root}/flash-linear-attention_amd/csrc', str(src), '-o', str(exe)], check=True)
    env = {k: v for k, v in os.environ.items() if k != 'LD_PRELOAD'}
    r = subprocess.run([str(exe)], capture_output=True, text=True, env=env)
    assert r.returncode == 0 and r.stdout == 'ok\n', r.stdout + r.stderr


class _Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: 0 if name.endswith('bytes') else self.calls.append(name) or 0


@pytest.fixture
def lib(monkeypatch):
    """The library is a stand-in that keeps record: nothing may be launched for a call that is refused."""
    from fla_hip import _lib
    from fla_hip.ops.attn import paged
    from fla_hip.ops.gated_delta_rule import _common
    lib = _Library()
    monkeypatch.setattr(_lib, 'load', lambda: lib)
    monkeypatch.setattr(_lib, 'host', lambda: _lib._PythonHost)
    monkeypatch.setattr(_common, 'current_device', lambda: None)
    monkeypatch.setattr(_common, 'current_stream_ptr', lambda dev: 0)
    monkeypatch.setattr(paged, 'require_gpu', lambda x, *_: x.device)
    return lib


def test_refusals(lib):
    a = _attn()
    c, t, n = torch.zeros(4, 8, 2, 16, dtype=BF), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    k, cos = torch.zeros(3, 5, 2, 16, dtype=BF), torch.zeros(9, 8)
    append = lambda k=k, v=k, kc=c, vc=c, t=t, n=n, **kw: a.paged_append(k, v, kc, vc, t, n, **kw)
    attn = lambda q=torch.zeros(3, 5, 4, 16, dtype=BF), kc=c, vc=c, t=t, n=n, **kw: a.paged_attn(q, kc, vc, t, n, **kw)
    keep = lambda kc=c, vc=c, t=t, n=n, rows=torch.zeros(3, 5, dtype=torch.int32), kept=n: a.paged_keep(kc, vc, t, n, rows, kept)
    append(), attn(), keep()
    assert lib.calls == ['gdn_paged_append', 'gdn_paged_attn', 'gdn_paged_keep']
    apart = c.transpose(2, 3).contiguous().transpose(2, 3)
    spread = c[:1].expand(4, 8, 2, 16)
    bad = [
        lambda: append(k=k[0]), lambda: append(v=k[:2]), lambda: append(k=k[:, :, :1], v=k[:, :, :1]), lambda: append(k=k.float(), v=k.float()), lambda: append(v=k.half()), lambda: append(kc=c[0], vc=c[0]),
        lambda: append(vc=c.half()), lambda: append(vc=c[:3]), lambda: append(t=t[:2]), lambda: append(t=t[0]), lambda: append(t=t.float()), lambda: append(n=n[:2]), lambda: append(n=n.float()),
        lambda: append(kc=apart, vc=apart), lambda: append(kc=spread), lambda: append(vc=spread), lambda: append(cos=cos), lambda: append(positions=torch.zeros(3, 5, dtype=torch.int32)),
        lambda: append(cos=cos, sin=cos, positions=torch.zeros(5, dtype=torch.int32)), lambda: append(q=k[:2]), lambda: append(q=k[..., :8]), lambda: append(q=k.float()),
        lambda: append(cos=torch.zeros(9, 9), sin=torch.zeros(9, 9)), lambda: append(cu_seqlens=torch.tensor([0, 5])), lambda: append(k=k[:1], v=k[:1], cu_seqlens=torch.tensor([0, 3, 2, 5])),
        lambda: append(kc=c[:, :0], vc=c[:, :0]),
        lambda: attn(q=torch.zeros(3, 5, 3, 16, dtype=BF)), lambda: attn(q=torch.zeros(3, 5, 4, 8, dtype=BF)), lambda: attn(q=torch.zeros(3, 5, 4, 16)), lambda: attn(q=torch.zeros(3, 4, 16, dtype=BF)),
        lambda: attn(kc=apart, vc=apart), lambda: attn(t=t[:2]), lambda: attn(n=n[:2]), lambda: attn(tree_mask=torch.zeros(5, 5)), lambda: attn(tree_mask=torch.zeros(4, 5, dtype=torch.bool)),
        lambda: attn(tree_mask=torch.zeros(2, 5, 5, dtype=torch.bool)), lambda: attn(tree_mask=torch.zeros(5, 0, dtype=torch.bool)), lambda: attn(cu_seqlens=torch.tensor([0, 5])),
        lambda: attn(q=torch.zeros(1, 5, 4, 16, dtype=BF), t=t[:1], n=n[:1], cu_seqlens=torch.tensor([0, 6])),
        lambda: attn(q=torch.zeros(1, 5, 4, 16, dtype=BF), t=t[:1], n=n[:1], cu_seqlens=torch.tensor([0, 5]), tree_mask=torch.zeros(1, 5, 5, dtype=torch.bool)),
        lambda: keep(rows=n), lambda: keep(kept=n[:2]), lambda: keep(rows=torch.zeros(3, 5)), lambda: keep(kept=n.float()), lambda: keep(kc=spread), lambda: keep(t=t[:1]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print('call', i)
    grad = [lambda: append(k=k.clone().requires_grad_()), lambda: append(kc=c.clone().requires_grad_()), lambda: attn(q=torch.zeros(3, 5, 4, 16, dtype=BF).requires_grad_()),
            lambda: keep(vc=c.clone().requires_grad_()), lambda: append(cos=cos.clone().requires_grad_(), sin=cos)]
    for call in grad:
        with pytest.raises(NotImplementedError):
            call()
    assert lib.calls == ['gdn_paged_append', 'gdn_paged_attn', 'gdn_paged_keep']
    with torch.no_grad():
        grad[0]()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(k, k)
        for call in (lambda: append(k=dual), lambda: attn(q=torch.cat([dual, dual], 2))):
            with pytest.raises(NotImplementedError):
                call()


def test_no_cpu_path():
    c = torch.zeros(1, 1, 1, 8, dtype=BF)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: _attn().paged_append(c, c, c, c, t, n), lambda: _attn().paged_attn(c, c, c, t, n), lambda: _attn().paged_keep(c, c, t, n, t, n)):
        with pytest.raises(RuntimeError, match='ROCm GPU'):
            call()


def test_library_refuses():
    import ctypes
    from fla_hip import _lib
    lib = _lib.load()

    def make(**kw):
        c = _lib.PagedCache(k=16, v=16, page_table=16, context=16, pages=2, page_size=4, heads=1, dim=16, table_cols=2, table_stride=2, dtype=0)
        for k, v in kw.items():
            setattr(c, k, v)
        return ctypes.byref(c)

    keep = lambda N=1, R=2, stride=2, rows=16, kept=16, **kw: lib.gdn_paged_keep(make(**kw), rows, stride, R, kept, N, None)
    invalid = [dict(pages=-1), dict(page_size=0), dict(heads=0), dict(dim=0), dict(table_cols=-1), dict(table_stride=1), dict(context=None), dict(k=None), dict(page_table=None), dict(N=-1), dict(R=-1),
               dict(stride=1), dict(rows=None), dict(kept=None), dict(N=65536)]
    assert [keep(**kw) for kw in invalid] == [_lib.GDN_ERR_INVALID] * len(invalid)
    unsupported = [dict(dtype=3), dict(pages=2 ** 31), dict(page_size=2 ** 31), dict(table_cols=2 ** 30, table_stride=2 ** 30)]
    assert [keep(**kw) for kw in unsupported] == [_lib.GDN_ERR_UNSUPPORTED] * len(unsupported)
    assert keep(N=0) == keep(R=0) == keep(pages=0, k=None, v=None) == _lib.GDN_OK
    attn = lambda cache=None, **kw: lib.gdn_paged_attn(make(**(cache or {})), ctypes.byref(_lib.PagedAttnCall(**{**dict(q=16, o=16, B=1, T=1, N=1, HQ=2, max_rows=1), **kw})), None, 0, None)
    invalid = [dict(B=-1), dict(T=-1), dict(HQ=-1), dict(N=2), dict(max_rows=-1), dict(q=None), dict(o=None), dict(cu_seqlens=16, B=2, N=2), dict(cu_seqlens=16, N=0), dict(cache=dict(heads=3), HQ=4)]
    assert [attn(**kw) for kw in invalid] == [_lib.GDN_ERR_INVALID] * len(invalid)
    assert attn(cache=dict(dtype=2)) == attn(cache=dict(dim=264)) == attn(cache=dict(dim=12)) == attn(cache=dict(page_size=2 ** 29 + 1)) == _lib.GDN_ERR_UNSUPPORTED
    assert attn() == _lib.GDN_ERR_WORKSPACE
    assert [attn(**kw) for kw in (dict(T=2 ** 25), dict(T=2 ** 26, HQ=1), dict(B=2 ** 40, N=2 ** 40), dict(T=2 ** 40))] == [_lib.GDN_ERR_UNSUPPORTED] * 4
    assert attn(B=0, N=0) == attn(T=0) == attn(HQ=0) == _lib.GDN_OK
    rows = lambda heads: ctypes.byref(_lib.RotaryRows(16, 16, heads))
    append = lambda k=1, v=1, q=None, cache=None, **kw: lib.gdn_paged_append(make(**(cache or {})), None if q is None else rows(q), rows(k), rows(v),
                                                                            ctypes.byref(_lib.RotaryCall(**{**dict(B=1, T=1, N=1, D=16, dtype=0, table_dtype=0), **kw})), None)
    invalid = [dict(k=2), dict(v=2), dict(D=8), dict(dtype=1, table_dtype=1), dict(q=-1), dict(cache=dict(page_size=0)), dict(rotary_dim=16)]
    assert [append(**kw) for kw in invalid] == [_lib.GDN_ERR_INVALID] * len(invalid)


@gpu
@pytest.mark.parametrize(('page_size', 'D', 'heads'), [(16, 128, 1), (4, 64, 5), (1, 576, 1)])
def test_keep_of_one_tensor_for_keys_and_values(page_size, D, heads):
    """Every slot is moved once: a path that shifts all of its rows by one or two, so that a row moved twice would have been the next."""
    N, R = 40, 33
    contexts = [(7 * n) % 50 for n in range(N)]
    lengths = [c + R for c in contexts]
    pages = pages_for(lengths, page_size)
    one, _ = cache(pages, page_size, heads, D, BF)
    t = table(lengths, page_size, pages)
    rows = torch.stack([torch.arange(R - 2) + 1 + n % 2 for n in range(N)]).int()
    want, now = one.clone().cpu(), one.cpu()
    for n in range(N):
        for i in range(R - 2):
            want[O.slot_of(t, n, contexts[n] + i, pages, page_size)] = now[O.slot_of(t, n, contexts[n] + int(rows[n, i]), pages, page_size)]
    _attn().paged_keep(one, one, t.to(DEV), torch.tensor(contexts, device=DEV), rows.to(DEV), torch.full((N,), R - 2, device=DEV))
    assert torch.equal(one.cpu(), want)
