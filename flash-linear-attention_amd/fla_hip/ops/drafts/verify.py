"""Verification of drafted tokens: which stand against the target's probabilities, and the token after them.  The count it returns is what the token recurrence takes as
``num_accepted_tokens`` (with a state per token), the path what ``fla_hip.ops.attn.paged_keep`` takes."""
from __future__ import annotations

import ctypes

import torch

from fla_hip import _lib
from fla_hip.ops.gated_delta_rule._common import as_index, dtype_code, launch, ptr, require_gpu, unit_rows


def verify_drafts(
    target_probs: torch.Tensor,
    draft_tokens: torch.Tensor,
    uniforms: torch.Tensor,
    parents: torch.Tensor | None = None,
    draft_probs: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Row 0 of a sequence is its last token, row r > 0 the draft ``draft_tokens[n, r]`` that follows row ``parents[n, r] < r`` (``[N, R]``, or ``[R]`` for all; default: a
    chain, the row before; a negative parent: no draft).  ``target_probs[n, r]`` (``[N, R, V]``) are the target's probabilities after row r, ``draft_probs[n, r]`` those that the
    drafts following row r were sampled from, in the same type (None: drafts that were not sampled).  ``uniforms [N, R]`` in [0, 1): entry r decides about draft r, entry 0
    draws the next token.  ``lengths [N]``: rows of a sequence (default R).

    From row 0 on the drafts that follow the row come to are asked in order: a draft x stands where ``u q(x) < p(x)``, and the walk goes on from it; one that does not
    leaves ``p = (p - q)+ / sum`` to the next (without draft_probs: p without x; p as it was where nothing would be left).  When none is left the next token is the first v
    with ``sum(p[: v + 1]) > u sum(p)``.  A draft outside the vocabulary (a padded row, -1) is passed over.  So tokens are distributed as the target's own, whatever was drafted.

    Returns ``(next_token [N] int64, num_accepted [N] int32, rows [N, R] int32)``: the token to go on with (-1 where p has no finite mass), the number of rows that stand, row 0
    among them, and which, in order, -1 behind them.  Computed in 64 bits; nothing of it is differentiable."""
    out = _lib.host().verify_drafts(target_probs, draft_tokens, uniforms, parents, draft_probs, lengths)
    if out is not None:
        return out
    dev = require_gpu(target_probs, draft_tokens, uniforms, *(t for t in (parents, draft_probs, lengths) if t is not None))
    if target_probs.dim() != 3 or target_probs.shape[1] < 1 or target_probs.shape[2] < 1:
        raise ValueError(f'target_probs must be [N, R, V], got {list(target_probs.shape)}')
    N, R, V = target_probs.shape
    if draft_probs is not None and (draft_probs.shape != target_probs.shape or draft_probs.dtype != target_probs.dtype):
        raise ValueError(f'draft_probs must be as target_probs {list(target_probs.shape)} {target_probs.dtype}, got {list(draft_probs.shape)} {draft_probs.dtype}')
    if tuple(uniforms.shape) != (N, R) or not uniforms.dtype.is_floating_point:
        raise ValueError(f'uniforms must be numbers in [0, 1) [{N}, {R}], got {list(uniforms.shape)} {uniforms.dtype}')
    code = dtype_code(target_probs.dtype)
    tokens = as_index(draft_tokens, dev, 'draft_tokens', (N, R))
    if uniforms.dtype == torch.float64:
        # (the nearest fp32 of a number below 1 may be 1)
        uniforms = uniforms.float().clamp(max=1 - 2.0 ** -24)
    uniforms = uniforms.detach().float().contiguous()
    if parents is not None:
        parents = as_index(parents, dev, 'parents', (R,) if parents.dim() == 1 else (N, R))
        parents = parents if parents.dtype == torch.int32 else parents.clamp(-1, R).int()
    if lengths is not None:
        lengths = as_index(lengths, dev, 'lengths', (N,))
        lengths = lengths if lengths.dtype == torch.int32 else lengths.clamp(0, R).int()
    p, q = unit_rows(target_probs.detach()), None if draft_probs is None else unit_rows(draft_probs.detach())
    token = torch.empty(N, dtype=torch.int64, device=dev)
    accepted = torch.empty(N, dtype=torch.int32, device=dev)
    rows = torch.empty(N, R, dtype=torch.int32, device=dev)
    call = _lib.DraftsCall(ptr(p), ptr(q), ptr(tokens), ptr(uniforms), ptr(parents), ptr(lengths), ptr(token), ptr(accepted), ptr(rows), (ctypes.c_int64 * 2)(*p.stride()[:2]),
                           (ctypes.c_int64 * 2)(*((0, 0) if q is None else q.stride()[:2])), 0 if parents is None or parents.dim() == 1 else R, N, R, V, code, code,
                           _lib.DRAFTS_TOKENS_INT64 if tokens.dtype == torch.int64 else 0)
    lib = _lib.load()
    need = lib.gdn_verify_drafts_workspace_bytes(ctypes.byref(call))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    launch(lib.gdn_verify_drafts, dev, ctypes.byref(call), ptr(ws), need)
    return token, accepted, rows
