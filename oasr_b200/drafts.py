"""Trees of drafted tokens: who sees whom, and which drafts stand (no reference operators).

A decoder that drafts several tokens a step hands the target model a tree of them: node 0 is the last token that stands, node
``i`` continues node ``parents[b, i] < i``; any other parent makes a node padding, and so what hangs on it.  A step:

    tree = draft_tree(parents)                                             # masks and depths
    ... every layer: qk_norm_rope at the positions length + tree.depth, write_kv_chunk at offset = length,
        fmha_tree(..., tree_mask=tree.mask, cache_seqlens=length + T) ...
    done = verify_drafts(logits, drafts, parents, uniforms)
    commit_drafts((k_pools, v_pools), block_table, length, done.path, done.counts)
    length += done.counts                                                   # done.tokens: the new tokens; the last one is node 0 of the next tree
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from . import _lib
from .attention import _index32, _narrow
from .functional import _dt, _one_device, _p, _stream


class DraftTree(NamedTuple):
    """What ``draft_tree`` returns."""

    mask: torch.Tensor
    depth: torch.Tensor


class VerifiedDrafts(NamedTuple):
    """What ``verify_drafts`` returns."""

    tokens: torch.Tensor
    path: torch.Tensor
    counts: torch.Tensor


def _whole32(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int32:
        if t.dtype != torch.int64:
            raise RuntimeError(f"{name} must be int32 or int64, got {t.dtype}")
        t = _narrow(t)
    return t if t.is_contiguous() else t.contiguous()


def draft_tree(parents: torch.Tensor) -> DraftTree:
    """``(mask, depth)`` of the trees ``parents (B, T)`` or of one tree ``(T,)``, T up to 1024.

    ``mask`` holds int32 words ``(..., T, ceil(T / 32))``: bit ``j % 32`` of word ``j // 32`` of row ``i`` is set where node ``j`` is ``i``
    itself or lies on its way from node 0, which is what ``fmha_tree`` takes.  ``depth (..., T)`` int32 counts the steps from node 0.
    Padding has no bits and depth -1."""
    if parents.dim() not in (1, 2):
        raise RuntimeError(f"parents must be (B, T) or (T,), got {tuple(parents.shape)}")
    parents = _whole32("parents", parents)
    _one_device(parents)
    T = parents.shape[-1]
    words = (T + 31) // 32
    mask = torch.empty(*parents.shape, words, dtype=torch.int32, device=parents.device)
    depth = torch.empty_like(parents)
    _lib.call("oasr_b200_draft_tree", mask.data_ptr(), depth.data_ptr(), parents.data_ptr(), parents.shape[0] if parents.dim() == 2 else 1, T,
              words, _stream(parents))
    return DraftTree(mask, depth)


def verify_drafts(logits: torch.Tensor, drafts: torch.Tensor, parents: torch.Tensor, uniforms: torch.Tensor, *,
                  temperature: Union[float, torch.Tensor] = 1.0, draft_probs: Optional[torch.Tensor] = None) -> VerifiedDrafts:
    """Which of the drafted tokens ``drafts (B, T)`` stand against the target's ``logits (B, T, V)``, and the token behind them.

    ``logits[b, i]`` is the target's row after node ``i`` of the tree ``parents (B, T)`` (``(T,)``: one for all); ``uniforms (B, T)`` fp32
    are random numbers of [0, 1).  The walk starts at node 0 with ``p = softmax(logits[b, n] / temperature)`` and tries the children ``c`` of
    ``n`` in order: with ``x = drafts[b, c]``, ``c`` is accepted iff ``uniforms[b, c] * q(x) < p(x)``, and the walk goes on from there; otherwise
    ``p`` becomes ``max(p - q, 0)``, normalised.  ``q`` is ``draft_probs[b, n]`` (fp32 ``(B, T, V)``: the distribution that all children of ``n``
    were drawn from, independently), or without it 1 at ``x``.  Where no child is accepted, the next token is the first whose cumulative ``p``
    passes ``uniforms[b, 0]``.  So the tokens are distributed as the target alone would draw them.  ``temperature`` is a number or ``(B,)``
    fp32; 0 or less (or NaN) is greedy: all of ``p`` on the first maximum.

    Returns int32 ``path (B, T)``, the nodes from node 0 on that stand, ``tokens (B, T)``, the token behind each of them (the last is the new
    one), both -1 behind the ``counts (B,)`` entries that they have: ``counts`` is how many tokens the step has brought and how many rows
    of the cache stay (``commit_drafts``).  A row of logits with a NaN, or whose maximum is not finite, ends the walk with token -1, and so do
    random numbers of 1 or more where nothing of ``p`` is left.  -inf logits are impossible tokens; a draft outside ``[0, V)`` is not accepted.

    Decisions are taken in 64 bits: weights to 2^-31, those below 2^-300 of the largest may be zeros.  The order of sums follows from the sizes of the call,
    so that the same call gives the same answer; a random number within some 2^-50 of a border may fall to either side of it in a batch of another size.
    Only rows on the accepted path are read."""
    shape = logits.shape
    if len(shape) != 3 or shape[2] < 1:
        raise RuntimeError(f"logits must be (B, T, V), got {tuple(shape)}")
    B, T, V = shape
    tree, one = (B, T), parents.dim() == 1
    if drafts.shape != tree or parents.shape != ((T,) if one else tree):
        raise RuntimeError(f"drafts must be ({B}, {T}) and parents ({B}, {T}) or ({T},), got {tuple(drafts.shape)} and {tuple(parents.shape)}")
    if uniforms.shape != tree or uniforms.dtype is not torch.float32:
        raise RuntimeError(f"uniforms must be fp32 ({B}, {T}), got {tuple(uniforms.shape)} {uniforms.dtype}")
    temperatures = None
    if isinstance(temperature, torch.Tensor):
        if temperature.shape != (B,) or temperature.dtype != torch.float32:
            raise RuntimeError(f"temperature must be a number or fp32 ({B},), got {tuple(temperature.shape)} {temperature.dtype}")
        temperatures, temperature = temperature if temperature.is_contiguous() else temperature.contiguous(), 1.0
    if draft_probs is not None and (draft_probs.shape != shape or draft_probs.dtype != torch.float32):
        raise RuntimeError(f"draft_probs must be fp32 {tuple(shape)}, got {tuple(draft_probs.shape)} {draft_probs.dtype}")
    drafts, parents = _whole32("drafts", drafts), _whole32("parents", parents)
    if not uniforms.is_contiguous():
        uniforms = uniforms.contiguous()
    _one_device(logits, drafts, parents, uniforms, temperatures, draft_probs)
    ls_b, ls_n, unit = logits.stride()
    if unit != 1 and V > 1:
        logits = logits.contiguous()
        ls_b, ls_n, _ = logits.stride()
    ps_b = ps_n = 0
    if draft_probs is not None:
        if draft_probs.stride(2) != 1 and V > 1:
            draft_probs = draft_probs.contiguous()
        ps_b, ps_n, _ = draft_probs.stride()
    device = logits.device
    tokens = torch.empty(tree, dtype=torch.int32, device=device)
    path = torch.empty_like(tokens)
    counts = torch.empty(B, dtype=torch.int32, device=device) if T else torch.zeros(B, dtype=torch.int32, device=device)
    _lib.call("oasr_b200_verify_drafts", tokens.data_ptr(), path.data_ptr(), counts.data_ptr(), logits.data_ptr(), ls_b, ls_n, drafts.data_ptr(),
              parents.data_ptr(), 0 if one else T, uniforms.data_ptr(), _p(draft_probs), ps_b, ps_n, _p(temperatures), temperature,
              B, T, V, _dt(logits), _stream(logits))
    return VerifiedDrafts(tokens, path, counts)
