"""Softmax attention of a serving step over a paged cache of keys and values: what the attention layers of a model that interleaves them with the gated delta
rule need beside the recurrence's pools of states.  (The reference keeps a cache of whole tensors, fla/layers/attn.py.)

The cache is ``k_cache, v_cache [pages, page_size, heads, dim]`` (any strides with a head's elements in a row); slot p of sequence n is slot ``p % page_size`` of page
``page_table[n, p // page_size]``.  ``context_lens [N]`` says how many slots hold a token before the step; row i of the step's tokens belongs to slot
``context_lens[n] + i``.  A step is ``paged_append``, then ``paged_attn``; with drafted tokens then ``fla_hip.ops.drafts.verify_drafts`` and ``paged_keep``,
after which ``context_lens`` grows by the number of rows that stand.  Lengths and tables stay on the GPU: no call waits for it, all can be captured in a graph."""
from __future__ import annotations

import ctypes

import torch

from fla_hip import _lib
from fla_hip.modules.rotary import check_tables, rotary_call, rows_of
from fla_hip.ops.gated_delta_rule._common import as_index, dtype_code, forward_only, launch, no_forward_mode, ptr, require_gpu, unit_rows, written
from fla_hip.ops.utils.index import check_cu_seqlens, max_seq_len


def _cache(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, context_lens: torch.Tensor, N: int, writes: bool) -> tuple:
    """The cache as the library takes it, and the tensors that have to live until the launch."""
    dev = k_cache.device
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError(f'k_cache and v_cache must be [pages, page_size, heads, dim] of one type, got {tuple(k_cache.shape)} {k_cache.dtype} and {tuple(v_cache.shape)} {v_cache.dtype}')
    pages, page_size, heads, dim = k_cache.shape
    if page_size < 1 or heads < 1 or dim < 1:
        raise ValueError(f'the cache has no slots: {tuple(k_cache.shape)}')
    for t in (k_cache, v_cache):
        if t.stride(3) != 1 and dim > 1:
            raise ValueError(f'{what} takes caches whose heads lie in a row, got strides {t.stride()}')
        if writes and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f'{what} writes into the cache, which must not overlap itself')
    if page_table.dim() != 2 or page_table.shape[0] != N:
        raise ValueError(f'page_table must be [{N}, pages of a sequence], got {list(page_table.shape)}')
    if page_table.dtype != torch.int32:
        # (a number that int32 cannot hold names no page either way)
        page_table = as_index(page_table, dev, 'page_table', page_table.shape).clamp(-1, 2 ** 31 - 1).int()
    table = unit_rows(page_table)
    if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        table = table.contiguous()
    context = as_index(context_lens, dev, 'context_lens', (N,))
    cache = _lib.PagedCache(ptr(k_cache), ptr(v_cache), ptr(table), ptr(context), (ctypes.c_int64 * 3)(*k_cache.stride()[:3]), (ctypes.c_int64 * 3)(*v_cache.stride()[:3]),
                            pages, page_size, heads, dim, table.shape[1], table.stride(0) if table.shape[0] > 1 else table.shape[1], dtype_code(k_cache.dtype),
                            int(context.dtype == torch.int32))
    return cache, (table, context)


def _sequences(x: torch.Tensor, cu_seqlens: torch.Tensor | None, max_seqlen: int | None) -> tuple:
    """(sequences, cu_seqlens as the kernels read it, rows of the longest); ``max_seqlen``: without a look at the boundaries."""
    B, T = x.shape[:2]
    if cu_seqlens is None:
        return B, None, T
    if B != 1:
        raise ValueError(f'The batch size is expected to be 1 rather than {B} when using `cu_seqlens`.')
    N = cu_seqlens.numel() - 1
    if N < 1:
        raise ValueError('cu_seqlens must hold N + 1 >= 2 boundaries')
    if max_seqlen is None:
        check_cu_seqlens(cu_seqlens, T)
        max_seqlen = max_seq_len(cu_seqlens)
    return N, as_index(cu_seqlens, x.device, 'cu_seqlens', (N + 1,)), max(0, min(int(max_seqlen), T))


def paged_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    max_seqlen: int | None = None,
    q: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    interleaved: bool = False,
) -> torch.Tensor | None:
    """The keys and values of a step's rows (k, v ``[B, T, heads, dim]``, or packed with ``cu_seqlens``) into their slots of the cache.  With ``cos`` and ``sin`` the keys are
    turned on the way (``fla_hip.modules.rotary_embedding``), and so are the queries ``q [B, T, query heads, dim]``, which are returned (None without q): at
    ``positions [B, T]``, by default the slot's number.  Rows whose slot has no page, and rows of no sequence, write nothing.  In the type of the cache; forward only.
    A page that is written belongs to one sequence."""
    done = _lib.host().paged_append(k, v, k_cache, v_cache, page_table, context_lens, cu_seqlens, max_seqlen, q, cos, sin, positions, interleaved)
    if done is not None:
        return done[0]
    dev = require_gpu(k, v, k_cache, v_cache, page_table, context_lens, *(t for t in (q, cos, sin, positions, cu_seqlens) if t is not None))
    if k.dim() != 4 or v.shape != k.shape or (q is not None and (q.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3])):
        raise ValueError(f'k and v must be [B, T, heads, dim] and q agree with them, got {tuple(k.shape)}, {tuple(v.shape)}' + ('' if q is None else f' and {tuple(q.shape)}'))
    if k.shape[2:] != k_cache.shape[2:]:
        raise ValueError(f'k has {list(k.shape[2:])} heads and elements, the cache {list(k_cache.shape[2:])}')
    if any(t is not None and t.dtype != k_cache.dtype for t in (k, v, q)):
        raise ValueError(f'k, v and q must be of the cache\'s type {k_cache.dtype}')
    if (cos is None) != (sin is None):
        raise ValueError('cos and sin come together')
    if positions is not None and cos is None:
        raise ValueError('positions are those of cos and sin')
    forward_only('paged_append', k, v, q, k_cache, v_cache, cos, sin)
    no_forward_mode('paged_append', k, v, q, k_cache, v_cache, cos, sin)
    N, cu, _ = _sequences(k, cu_seqlens, max_seqlen)
    cache, held = _cache('paged_append', k_cache, v_cache, page_table, context_lens, N, True)
    if cos is not None:
        cos, sin = check_tables(k, cos, sin)
    if positions is not None:
        positions = as_index(positions, dev, 'positions', k.shape[:2])
    k, v, q = unit_rows(k), unit_rows(v), None if q is None else unit_rows(q)
    out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=dev)
    call = rotary_call(k, cos, sin, interleaved, False, positions, None, 0, cu)
    launch(_lib.load().gdn_paged_append, dev, ctypes.byref(cache), None if q is None else ctypes.byref(rows_of(q, out)), ctypes.byref(rows_of(k, None)),
           ctypes.byref(rows_of(v, None)), ctypes.byref(call))
    del held
    written(k_cache, v_cache)
    return out


def paged_attn(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    tree_mask: torch.Tensor | None = None,
    scale: float | None = None,
    cu_seqlens: torch.Tensor | None = None,
    max_seqlen: int | None = None,
) -> torch.Tensor:
    """Attention of a step's rows, whose keys and values are in the cache by then: q ``[B, T, query heads, dim]`` (a multiple of the cache's heads; head h reads the cache's
    head ``h // group``) or packed with ``cu_seqlens``.  A row sees the whole context and, of the step's own rows, itself and those before it, or what ``tree_mask`` says:
    truth values ``[T, columns]`` (one tree for all), ``[B, T, columns]``, or ``[rows, columns]`` of a packed batch; row i sees row j of its sequence where ``tree_mask[.., i, j]``,
    columns that are missing are not seen.  A row that sees nothing, and one of no sequence, gets 0.  ``scale``: default ``dim ** -0.5``.  ``max_seqlen`` (packed): at
    least the longest sequence's rows, then the boundaries are not read by the host.  bf16 or fp16, dim a multiple of 8 up to 256; forward only."""
    o = _lib.host().paged_attn(q, k_cache, v_cache, page_table, context_lens, tree_mask, scale, cu_seqlens, max_seqlen)
    if o is not None:
        return o
    dev = require_gpu(q, k_cache, v_cache, page_table, context_lens, *(t for t in (tree_mask, cu_seqlens) if t is not None))
    if q.dim() != 4 or k_cache.dim() != 4 or q.shape[3] != k_cache.shape[3]:
        raise ValueError(f'q must be [B, T, heads, dim] with the dim of the cache, got {tuple(q.shape)} and {tuple(k_cache.shape)}')
    if k_cache.shape[2] < 1 or q.shape[2] % k_cache.shape[2]:
        raise ValueError(f'the queries\' heads ({q.shape[2]}) must be a multiple of the cache\'s ({k_cache.shape[2]})')
    if q.dtype != k_cache.dtype:
        raise ValueError(f'q must be of the cache\'s type {k_cache.dtype}, got {q.dtype}')
    forward_only('paged_attn', q, k_cache, v_cache)
    no_forward_mode('paged_attn', q, k_cache, v_cache)
    B, T, HQ, D = q.shape
    N, cu, longest = _sequences(q, cu_seqlens, max_seqlen)
    cache, held = _cache('paged_attn', k_cache, v_cache, page_table, context_lens, N, False)
    seq_stride = row_stride = cols = 0
    if tree_mask is not None:
        if tree_mask.dtype != torch.bool:
            raise ValueError(f'tree_mask must hold truth values, got {tree_mask.dtype}')
        shapes = ('T', ) if cu is not None else ('T', 'B, T')
        if not (tree_mask.dim() == 2 and tree_mask.shape[0] == T) and not (cu is None and tree_mask.dim() == 3 and tree_mask.shape[:2] == (B, T)):
            raise ValueError(f'tree_mask must be ' + ' or '.join(f'[{s}, columns]' for s in shapes) + f' with B = {B}, T = {T}, got {list(tree_mask.shape)}')
        tree_mask = unit_rows(tree_mask)
        cols, row_stride, seq_stride = tree_mask.shape[-1], tree_mask.stride(-2), tree_mask.stride(0) if tree_mask.dim() == 3 else 0
    q = unit_rows(q)
    o = torch.empty(B, T, HQ, D, dtype=q.dtype, device=dev)
    call = _lib.PagedAttnCall(ptr(q), ptr(o), ptr(cu), ptr(tree_mask) if cols else None, (ctypes.c_int64 * 3)(*q.stride()[:3]), seq_stride, row_stride, cols, B, T, N, HQ,
                              longest, D ** -0.5 if scale is None else scale, _lib.FLAG_CU_INT32 if cu is not None and cu.dtype == torch.int32 else 0)
    if tree_mask is not None and not cols:
        raise ValueError('tree_mask has no columns')
    lib = _lib.load()
    need = lib.gdn_paged_attn_workspace_bytes(ctypes.byref(cache), ctypes.byref(call))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    launch(lib.gdn_paged_attn, dev, ctypes.byref(cache), ctypes.byref(call), ptr(ws), need)
    del held
    return o


def paged_keep(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    rows: torch.Tensor,
    num_kept: torch.Tensor,
) -> None:
    """The rows of a step that stand, moved to the front of its slots: slot ``context_lens[n] + i`` becomes what slot ``context_lens[n] + rows[n, i]`` was, for
    ``i < num_kept[n]`` (rows ``[N, R]`` int32 with ``rows[n, i] >= i``, num_kept ``[N]``: the path and the count that ``verify_drafts`` returns).  Any other entry, and one whose
    slots have no page, leaves its slot as it is.  k_cache and v_cache may be one tensor.  The positions that keys were turned by stay: a node of a tree is at the same depth before and after."""
    if _lib.host().paged_keep(k_cache, v_cache, page_table, context_lens, rows, num_kept) is not None:
        return
    dev = require_gpu(k_cache, v_cache, page_table, context_lens, rows, num_kept)
    if rows.dim() != 2:
        raise ValueError(f'rows must be [N, R], got {list(rows.shape)}')
    forward_only('paged_keep', k_cache, v_cache)
    no_forward_mode('paged_keep', k_cache, v_cache)
    N, R = rows.shape
    cache, held = _cache('paged_keep', k_cache, v_cache, page_table, context_lens, N, True)
    # (a number that int32 cannot hold names no row, a larger count is held to R either way)
    rows, kept = (t if t.dtype == torch.int32 else t.clamp(-1, 2 ** 31 - 1).int()
                  for t in (as_index(rows, dev, 'rows', (N, R)), as_index(num_kept, dev, 'num_kept', (N,))))
    launch(_lib.load().gdn_paged_keep, dev, ctypes.byref(cache), ptr(rows), R, R, ptr(kept), N)
    del held
    written(k_cache, v_cache)
