"""Rotary positions, with the names of the reference's fla/modules/rotary.py: ``rotary_embedding`` (differentiable) and ``RotaryEmbedding``; ``rotary_embedding_qk``
turns queries and keys in one launch.  All compute is done by ``gdn_rotary`` of the HIP library; the tables are made once, by torch.

The tables are kept in fp32 from angles in 64 bits (the reference keeps them in the rows' type, from angles in 32): at position 100000 the fastest pair's angle is then
right to 1e-11 instead of 4e-3.  Tables of the rows' type are taken as well."""
from __future__ import annotations

import ctypes
import math

import torch
import torch.nn as nn

from fla_hip import _lib
from fla_hip.ops.gated_delta_rule._common import as_index, dtype_code, forward_only, launch, no_forward_mode, ptr, require_gpu, unit_rows, written
from fla_hip.ops.utils.index import check_cu_seqlens, max_seq_len


def rows_of(x: torch.Tensor, y: torch.Tensor | None) -> _lib.RotaryRows:
    return _lib.RotaryRows(ptr(x), ptr(y), x.shape[2], (ctypes.c_int64 * 3)(*x.stride()[:3]), (ctypes.c_int64 * 3)(*(y if y is not None else x).stride()[:3]))


def check_tables(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """cos, sin ``[positions, R / 2]`` of one type, x's or fp32, their rows equally far apart."""
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise ValueError(f'cos and sin must be [positions, rotary_dim / 2], got {tuple(cos.shape)} and {tuple(sin.shape)}')
    if cos.shape[1] == 0 or 2 * cos.shape[1] > x.shape[-1]:
        raise ValueError(f'cos and sin turn {2 * cos.shape[1]} elements of heads of {x.shape[-1]}')
    if cos.dtype != sin.dtype or cos.dtype not in (x.dtype, torch.float32):
        cos, sin = cos.float(), sin.float()
    return table_rows(cos, sin)


def table_rows(cos: torch.Tensor, sin: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The tables with their rows equally far apart, a row's elements side by side."""
    cos, sin = unit_rows(cos), unit_rows(sin)
    if cos.stride(0) != sin.stride(0) or cos.stride(0) < cos.shape[1]:
        cos, sin = cos.contiguous(), sin.contiguous()
    return cos, sin


def as_saved(x: torch.Tensor | None, dtype: torch.dtype, shape, device: torch.device) -> torch.Tensor | None:
    """A saved tensor in the type and the place that it had (saved-tensor hooks may hand back others)."""
    if x is None:
        return None
    if x.shape != shape:
        raise ValueError(f'a saved tensor {tuple(shape)} came back as {tuple(x.shape)}')
    return x.to(device=device, dtype=dtype)


def rotary_call(x: torch.Tensor, cos: torch.Tensor | None, sin: torch.Tensor | None, interleaved: bool, back: bool, positions: torch.Tensor | None,
                offsets: torch.Tensor | None, offset: int, cu_seqlens: torch.Tensor | None) -> _lib.RotaryCall:
    """Everything of a call but its tensors; the indices are as ``as_index`` leaves them."""
    B, T, _, D = x.shape
    call = _lib.RotaryCall(ptr(cos), ptr(sin), ptr(positions), ptr(offsets), ptr(cu_seqlens), B=B, T=T, D=D, offset=offset,
                           N=B if cu_seqlens is None else cu_seqlens.numel() - 1, dtype=dtype_code(x.dtype))
    if cos is not None:
        call.table_rows, call.table_stride, call.rotary_dim, call.table_dtype = cos.shape[0], cos.stride(0), 2 * cos.shape[1], dtype_code(cos.dtype)
    else:
        call.table_dtype = call.dtype
    flags = (_lib.ROTARY_INTERLEAVED if interleaved else 0) | (_lib.ROTARY_BACK if back else 0)
    for t, flag in ((positions, _lib.ROTARY_POSITIONS_INT32), (offsets, _lib.ROTARY_OFFSETS_INT32), (cu_seqlens, _lib.FLAG_CU_INT32)):
        if t is not None and t.dtype == torch.int32:
            flags |= flag
    call.flags = flags
    return call


def _turn(xs: tuple, cos, sin, interleaved, back, positions, offsets, offset, cu_seqlens, inplace: bool) -> tuple:
    xs = tuple(unit_rows(x) for x in xs)
    ys = xs if inplace else tuple(torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs)
    call = rotary_call(xs[0], cos, sin, interleaved, back, positions, offsets, offset, cu_seqlens)
    rows = (_lib.RotaryRows * len(xs))(*(rows_of(x, y) for x, y in zip(xs, ys)))
    launch(_lib.load().gdn_rotary, xs[0].device, rows, len(xs), ctypes.byref(call))
    return ys


class RotaryFunction(torch.autograd.Function):
    """A turn by the tables' angles; its gradient is the turn back, which is this function again (and so differentiable itself)."""

    # (the rows first: of a view that is written torch takes the gradient's way through the first operand)
    @staticmethod
    def forward(ctx, a, b, cos, sin, interleaved, back, positions, offsets, offset, cu_seqlens, inplace):
        xs = (a,) if b is None else (a, b)
        ctx.save_for_backward(cos, sin, positions, offsets, cu_seqlens)
        ctx.call = (interleaved, back, offset)
        ctx.saved_as = [None if t is None else (t.dtype, t.shape, t.device) for t in (cos, sin, positions, offsets, cu_seqlens)]
        ctx.dtype = xs[0].dtype
        ctx.set_materialize_grads(False)
        if inplace:
            ctx.mark_dirty(*xs)
        return _turn(xs, cos, sin, interleaved, back, positions, offsets, offset, cu_seqlens, inplace)

    @staticmethod
    def backward(ctx, *dys):
        interleaved, back, offset = ctx.call
        cos, sin, positions, offsets, cu_seqlens = (t if was is None else as_saved(t, *was) for t, was in zip(ctx.saved_tensors, ctx.saved_as))
        cos, sin = table_rows(cos, sin)
        positions, offsets, cu_seqlens = (None if t is None else t.contiguous() for t in (positions, offsets, cu_seqlens))
        at = [i for i, dy in enumerate(dys) if dy is not None]
        dxs = [None, None]
        if at:
            turned = [dys[i].to(ctx.dtype) for i in at] + [None]
            grads = RotaryFunction.apply(*turned[:2], cos, sin, interleaved, not back, positions, offsets, offset, cu_seqlens, False)
            for i, dx in zip(at, grads):
                dxs[i] = dx
        return (*dxs, *(None,) * 9)


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one type share an element: whether sum i s - sum j r is the distance of their first elements for some indices i, j within their sizes."""
    if not a.numel() or not b.numel():
        return False
    spans = {}                                                        # stride -> least and largest number of steps
    for x, sign in ((a, 1), (b, -1)):
        for size, stride in zip(x.shape, x.stride()):
            if size > 1 and stride:
                low, high = spans.get(stride, (0, 0))
                spans[stride] = (low, high + size - 1) if sign > 0 else (low - (size - 1), high)
    steps = sorted(((s, *lh) for s, lh in spans.items()), reverse=True)
    inner = [(0, 0)]                                                  # what the strides behind reach
    for s, low, high in reversed(steps):
        inner.insert(0, (inner[0][0] + s * low, inner[0][1] + s * high))
    left = 10000

    def reached(distance: int, at: int) -> bool:
        nonlocal left
        left -= 1
        if left < 0:                                                  # (strides that fold into each other many times: taken for an overlap)
            return True
        if at == len(steps):
            return distance == 0
        s, low, high = steps[at]
        behind = inner[at + 1]
        return any(reached(distance - n * s, at + 1) for n in range(max(low, -((behind[1] - distance) // s)), min(high, (distance - behind[0]) // s) + 1))

    return reached((b.data_ptr() - a.data_ptr()) // a.element_size(), 0)


def check_written(x: torch.Tensor) -> None:
    """What torch refuses to have written in place, before it is written (an autograd function says so when its forward has run)."""
    if not x.requires_grad:
        return
    if x.is_leaf or (x._is_view() and x._base.is_leaf and x._base.requires_grad):
        raise RuntimeError('inplace=True: a leaf that requires a gradient, or a view of one, cannot be turned in place')
    if x._is_view() and torch._C._autograd._get_creation_meta(x) != torch._C._autograd.CreationMeta.DEFAULT:
        raise RuntimeError('inplace=True: a view that came with others (split, unbind), or was made without a graph, cannot be turned in place: slice the tensor, or turn it out of place')


def _rotary(xs: tuple, cos, sin, interleaved, inplace, seqlen_offsets, cu_seqlens, max_seqlen, positions) -> tuple:
    if not inplace:
        ys = _lib.host().rotary(xs[0], xs[1] if len(xs) > 1 else None, cos, sin, interleaved, seqlen_offsets, cu_seqlens, max_seqlen, positions)
        if ys is not None:
            return ys
    x = xs[0]
    dev = require_gpu(*xs, cos, sin)
    for other in xs:
        if other.dim() != 4:
            raise ValueError(f'rotary positions take [B, T, heads, dim], got {tuple(other.shape)}')
        if other.shape[:2] != x.shape[:2] or other.shape[3] != x.shape[3] or other.dtype != x.dtype:
            raise ValueError(f'queries and keys must agree in batch, length, head size and type, got {tuple(x.shape)} {x.dtype} and {tuple(other.shape)} {other.dtype}')
    dtype_code(x.dtype)
    cos, sin = check_tables(x, cos, sin)
    forward_only('a gradient of the tables of rotary positions', cos, sin)
    no_forward_mode('rotary positions', *xs, cos, sin)
    B, T = x.shape[:2]
    N, longest = B, T if max_seqlen is None or cu_seqlens is None else max_seqlen
    if cu_seqlens is not None:
        if B != 1:
            raise ValueError(f'The batch size is expected to be 1 rather than {B} when using `cu_seqlens`.')
        N = cu_seqlens.numel() - 1
        if N < 1:
            raise ValueError('cu_seqlens must hold N + 1 >= 2 boundaries')
        if max_seqlen is None:
            check_cu_seqlens(cu_seqlens, T)
            longest = max_seq_len(cu_seqlens)
        cu_seqlens = as_index(cu_seqlens, dev, 'cu_seqlens', (N + 1,))
    offsets, offset = None, 0
    if positions is not None:
        positions = as_index(positions, dev, 'positions', (B, T))
        if isinstance(seqlen_offsets, torch.Tensor) or seqlen_offsets:
            raise ValueError('positions take the place of seqlen_offsets: give one of the two')
    elif isinstance(seqlen_offsets, torch.Tensor):
        offsets = as_index(seqlen_offsets, dev, 'seqlen_offsets', (N,))
    else:
        offset = int(seqlen_offsets)
        if offset < 0 or offset + longest > cos.shape[0]:
            raise ValueError(f'the tables have {cos.shape[0]} positions, positions {offset} to {offset + longest - 1} are needed')
    if inplace:
        for x in xs:
            if x.stride(-1) != 1 and x.shape[-1] > 1:
                raise ValueError('inplace=True needs heads whose elements lie in a row')
            if any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
                raise ValueError('inplace=True needs a tensor that does not overlap itself')
        if len(xs) == 2 and overlap(*xs):
            raise ValueError('inplace=True needs queries and keys that do not overlap')
    if torch.is_grad_enabled() and any(x.requires_grad for x in xs):
        if inplace:
            for x in xs:
                check_written(x)
            if len(xs) == 2 and not all(x.requires_grad and not x._is_view() for x in xs):
                # (torch writes into a view for a function of one result only; a tensor without a gradient stays one)
                return sum((_rotary((x,), cos, sin, interleaved, True, offset if offsets is None else offsets, cu_seqlens, max_seqlen, positions) for x in xs), ())
        return RotaryFunction.apply(*(*xs, None)[:2], cos, sin, interleaved, False, positions, offsets, offset, cu_seqlens, inplace)
    ys = _turn(tuple(x.detach() for x in xs), cos, sin, interleaved, False, positions, offsets, offset, cu_seqlens, inplace)
    if inplace:
        written(*xs)
        return xs
    return ys


def rotary_embedding(
    x: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    interleaved: bool = False,
    inplace: bool = False,
    seqlen_offsets: int | torch.Tensor = 0,
    cu_seqlens: torch.Tensor | None = None,
    max_seqlen: int | None = None,
    positions: torch.Tensor | None = None,
) -> torch.Tensor:
    """x ``[B, T, H, D]`` turned by the angles of its positions: ``(x1 cos - x2 sin, x1 sin + x2 cos)`` for the pairs ``(j, j + R/2)``, or ``(2j, 2j + 1)`` with
    ``interleaved``; cos, sin ``[positions, R/2]``, elements behind R pass through.  Row i of a sequence is at position ``i + seqlen_offsets`` (a number, or
    ``[N]``), or at ``positions [B, T]``.  ``cu_seqlens [N + 1]``: a packed batch; with ``max_seqlen`` (at least the longest sequence) its boundaries are not read by the host.
    A position that only the GPU knows and the tables do not have gives NaN; rows of no sequence are handed on as they are.  Differentiable in x, any number of times."""
    return _rotary((x,), cos, sin, interleaved, inplace, seqlen_offsets, cu_seqlens, max_seqlen, positions)[0]


def rotary_embedding_qk(
    q: torch.Tensor,
    k: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    interleaved: bool = False,
    inplace: bool = False,
    seqlen_offsets: int | torch.Tensor = 0,
    cu_seqlens: torch.Tensor | None = None,
    max_seqlen: int | None = None,
    positions: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``rotary_embedding`` of queries and keys (of their own numbers of heads) in one launch."""
    return _rotary((q, k), cos, sin, interleaved, inplace, seqlen_offsets, cu_seqlens, max_seqlen, positions)


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """(angles per position of the ``dim / 2`` pairs in 64 bits, factor of cos and sin).  ``scaling``: ``{'type': 'linear' | 'ntk' | 'yarn', 'factor': s, ...}`` for
    contexts s times the trained one - every angle divided by s; the base times ``s ** (dim / (dim - 2))``; or (with ``original_max_position_embeddings``, and
    ``beta_fast`` 32, ``beta_slow`` 1, ``attention_factor`` 0.1 ln s + 1) the pairs that turn less than beta_slow times in the trained context divided by s, those that
    turn more than beta_fast times left alone, and in between a ramp.  Any other entry raises: it would make other tables than its model's."""
    if dim <= 0 or dim % 2:
        raise ValueError(f'the turned part of a head must be even, got {dim}')
    inverse = lambda b: b ** (-torch.arange(0, dim, 2, dtype=torch.float64, device='cpu') / dim)
    if scaling is None:
        return inverse(base), 1.0
    kind, factor = scaling.get('type', scaling.get('rope_type')), float(scaling['factor'])
    if scaling.get('rope_type', kind) != kind:
        raise ValueError(f"scaling is of type {kind!r} and of rope_type {scaling['rope_type']!r}")
    taken = {'type', 'rope_type', 'factor', 'original_max_position_embeddings'} | ({'beta_fast', 'beta_slow', 'attention_factor'} if kind == 'yarn' else set())
    if set(scaling) - taken:
        raise ValueError(f'scaling of type {kind!r} takes {sorted(taken)}, got {sorted(set(scaling) - taken)} besides')
    if not factor >= 1:
        raise ValueError(f'the factor of a scaled context must be at least 1, got {factor}')
    if kind == 'linear':
        return inverse(base) / factor, 1.0
    if kind == 'ntk':
        if dim <= 2:
            raise ValueError('scaling by the base needs more than one pair')
        return inverse(base * factor ** (dim / (dim - 2))), 1.0
    if kind == 'yarn':
        trained = scaling['original_max_position_embeddings']
        at = lambda turns: dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(at(scaling.get('beta_fast', 32))), 0)
        high = min(math.ceil(at(scaling.get('beta_slow', 1))), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64, device='cpu') - low) / max(high - low, 1e-3)).clamp(0, 1)
        inv = inverse(base)
        return inv / factor * ramp + inv * (1 - ramp), float(scaling.get('attention_factor', 0.1 * math.log(factor) + 1.0))
    raise ValueError(f"scaling must be of type 'linear', 'ntk' or 'yarn', got {kind!r}")


class RotaryEmbedding(nn.Module):
    """Queries and keys turned by their positions (``fla.modules.RotaryEmbedding``), ``dim`` elements of each head.  ``scale_base``: the turned pairs of queries are scaled by
    ``s ** ((t - c) / scale_base)``, those of keys by its inverse, ``s = (2j + 0.4 dim) / (1.4 dim)``.  c is ``scale_center``; without one it is the middle ``T // 2`` of the call's
    positions, which holds for whole sequences only: the scales of keys from one call and queries of another would not cancel, so calls that go on from others
    (``seqlen_offset``, ``positions``) raise.  ``scaling``: see ``rotary_frequencies``.  The tables grow with the positions asked for and are no part of the state; those that a
    captured graph reads are kept as long as the module."""

    def __init__(self, dim: int, base: float = 10000.0, scale_base: float | None = None, interleaved: bool = False, pos_idx_in_fp32: bool = True,
                 device: torch.device | None = None, scaling: dict | None = None, scale_center: int | None = None):
        super().__init__()
        if not pos_idx_in_fp32:
            raise NotImplementedError('angles are formed in 64 bits: pos_idx_in_fp32=False is not offered')
        if scale_center is not None and scale_base is None:
            raise ValueError('scale_center is that of scale_base')
        self.dim, self.base, self.scale_base, self.interleaved, self.scaling, self.scale_center = dim, float(base), scale_base, interleaved, scaling, scale_center
        self._prefixes = scale_base is None or scale_center is not None      # (tables of more positions begin with those of fewer)
        self._frequencies, self.attention_factor = rotary_frequencies(dim, self.base, scaling)
        # (the reference's buffer, for who reads it: the tables are made from the frequencies in 64 bits)
        self.register_buffer('inv_freq', self._frequencies.float().to(torch.get_default_device() if device is None else device), persistent=False)
        self._tables, self._captured = None, []

    def extra_repr(self) -> str:
        return f'dim={self.dim}, base={self.base}, interleaved={self.interleaved}' + (f', scale_base={self.scale_base}' if self.scale_base is not None else '') + (
            f', scale_center={self.scale_center}' if self.scale_center is not None else '') + (
            f', scaling={self.scaling}' if self.scaling is not None else '')

    def tables(self, positions: int, device: torch.device) -> tuple[torch.Tensor, ...]:
        """cos, sin for at least this many positions (and, with ``scale_base``, the keys' cos, sin), fp32."""
        device = torch.device(device)
        kept, captured = self._tables, device.type == 'cuda' and torch.cuda.is_current_stream_capturing()
        if kept is not None and kept[0].device == device and (kept[0].shape[0] >= positions if self._prefixes else kept[0].shape[0] == positions):
            if captured and not any(t is kept for t in self._captured):
                self._captured.append(kept)
            return kept
        if captured:
            raise RuntimeError(f'the tables of {positions} positions are not made yet: call RotaryEmbedding.tables({positions}, device) before the capture')
        center = positions // 2 if self.scale_center is None else self.scale_center
        if self.scale_base is not None:
            # ((2/7) ** (distance / scale_base) and its inverse are normal numbers of fp32)
            reach = int(126 * abs(self.scale_base) / math.log2(3.5))
            most = center + reach + 1
            if positions > most or center > reach:
                raise ValueError(f'scales of positions more than {reach} from their centre {center} leave the range of fp32: {positions} positions were asked for')
        if kept is not None and kept[0].device == device and self._prefixes:
            # (asked for position after position: seldom made)
            positions = max(positions, 2 * kept[0].shape[0] if self.scale_base is None else min(2 * kept[0].shape[0], most))
        if kept is not None and kept[0].is_cuda:
            torch.cuda.synchronize(kept[0].device)                       # (a call on another stream may still read those that go)
        # Made on the host (whatever the default device) and copied while it waits: whatever stream reads them, they are there.
        with torch.no_grad(), torch.inference_mode(False):
            t = torch.arange(positions, dtype=torch.float64, device='cpu')
            angle = t[:, None] * self._frequencies
            cos, sin = angle.cos() * self.attention_factor, angle.sin() * self.attention_factor
            if self.scale_base is None:
                tables = (cos, sin)
            else:
                s = (torch.arange(0, self.dim, 2, dtype=torch.float64, device='cpu') + 0.4 * self.dim) / (1.4 * self.dim)
                scale = s ** ((t - center) / self.scale_base)[:, None]
                tables = (cos * scale, sin * scale, cos / scale, sin / scale)
            self._tables = tuple(x.float().to(device) for x in tables)
        return self._tables

    def forward(
        self,
        q: torch.Tensor,
        k: torch.Tensor,
        seqlen_offset: int | torch.Tensor = 0,
        cu_seqlens: torch.Tensor | None = None,
        max_seqlen: int | None = None,
        positions: torch.Tensor | None = None,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """q, k ``[B, T, heads, D]``.  Where positions are known to the GPU alone (``seqlen_offset`` or ``positions`` a tensor) ``max_seqlen`` says how many the tables
        have to have."""
        known = not isinstance(seqlen_offset, torch.Tensor) and positions is None
        if not known and max_seqlen is None:
            raise ValueError('max_seqlen is needed where seqlen_offset or positions are tensors: the number of positions that the tables have to have')
        if not self._prefixes and (not known or int(seqlen_offset)):
            raise ValueError('scales around the middle of a call do not cancel between calls: give RotaryEmbedding a scale_center for calls that go on from others')
        count = (max_seqlen if max_seqlen is not None else q.shape[1]) + (int(seqlen_offset) if known else 0)
        tables = self.tables(count, q.device)
        call = dict(interleaved=self.interleaved, seqlen_offsets=seqlen_offset, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen if cu_seqlens is not None else None, positions=positions)
        if self.scale_base is None:
            return rotary_embedding_qk(q, k, *tables, **call)
        return rotary_embedding(q, *tables[:2], **call), rotary_embedding(k, *tables[2:], **call)
