"""Attention of drafted tokens over a key/value cache, and the trees between them.

A step hands the model T drafted tokens per sequence instead of one: the last accepted token (node 0, the root) and guesses
that continue it, each with a parent among the nodes before it.  Node t lies in slot ``pos + t`` of the cache; it sees what was
accepted (slots before ``pos``), itself and its ancestors.  With one token per sequence this is ordinary decoding, over caches
of 8 bits too.

Reference semantics: blockwise attention with (m, s, acc) merging and grouped query heads
(compiler/mesh_compiler/operations.py:7072-7166).
"""
from __future__ import annotations

import struct

import torch

from .. import _native
from .cache import KVCache, _ints, _launch, _lib

MAX_DRAFTS = 64
# ``MeshDraftAttention`` (csrc/ops/draft_api.h): q, out, their strides, pos, counts, visible, T, q_heads, window, splits, scale, scratch, status
_ARGS = struct.Struct("@PPqqqqPPPiiiifPP")


def tree_visible(parents) -> torch.Tensor:
    """``parents [B, T]`` (a list or an integer tensor; ``parents[b][t] < t``, negative: no parent) -> int64 ``[B, T]`` on the host: bit j
    of a node's word is set for itself and its ancestors.  A tree that does not change is turned into words once."""
    rows = parents.tolist() if isinstance(parents, torch.Tensor) else parents
    words = []
    for row in rows:
        if len(row) > MAX_DRAFTS:
            raise ValueError(f"tree_visible: at most {MAX_DRAFTS} drafts, got {len(row)}")
        seen: list[int] = []
        for t, p in enumerate(row):
            if p >= t:
                raise ValueError(f"tree_visible: node {t} has parent {p}; a parent comes before its children")
            seen.append((seen[p] if p >= 0 else 0) | 1 << t)
        words.append([w - (1 << 64) if w >> 63 else w for w in seen])
    return torch.tensor(words, dtype=torch.int64).reshape(len(rows), len(words[0]) if words else 0)


def tree_depth(visible: torch.Tensor) -> torch.Tensor:
    """Depth of every node (the root: 0) from its word, int32: its position is ``pos`` plus this."""
    bits = torch.arange(64, device=visible.device)
    return (((visible[..., None] >> bits) & 1).sum(-1).clamp(min=1) - 1).to(torch.int32)


def _overlap(strides, B: int, T: int, row: int) -> bool:
    """Whether rows [b, t] of `row` values may meet."""
    (s1, n1), (s2, n2) = sorted(((strides[0], B), (strides[1], T)))
    return (n1 > 1 and s1 < row) or (n2 > 1 and s2 < (n1 - 1) * s1 + row)


def draft_attention(q: torch.Tensor, cache: KVCache, pos: torch.Tensor, *, counts: torch.Tensor | None = None,
                    visible: torch.Tensor | None = None, window: int = 0, scale: float | None = None,
                    out: torch.Tensor | None = None, splits: int = 0) -> torch.Tensor:
    """``q [B, T, q_heads, head_dim]`` bf16 (heads dense, T <= 64) against ``cache`` -> ``out`` of the same shape.

    ``pos [B]`` int32: slots before it are seen by every node (with ``window``: those less than ``window`` positions back; a
    node's position is ``pos`` plus the bits set in its word, less one); node t lies in slot ``pos[b] + t``, where
    :meth:`KVCache.append` has put it.  ``visible [B, T]`` int64: bit j says that the node sees node j (``None``: the ones before it and itself);
    ``counts [B]`` int32: nodes of each sequence (``None``: T); later ones are neither computed nor written.  A node that
    sees nothing gets zeros.  ``out`` may be ``q``, but must not meet it otherwise.  A ``window`` must not be shorter than T.
    ``splits``: CTAs among which the keys of all sequences are shared out, in equal shares (0: what pays for these sizes).

    Sums of the softmax are fp32; its weights are rounded to fp16 (8-bit rows) or bf16 (bf16 rows, half a step of the result's own type;
    ``ops.decode.DecodeAttention`` over the same rows keeps them in fp32) before the second product."""
    B, H, S, hd = cache.k.shape
    dev, bf16 = cache.device, torch.bfloat16
    shape = q.shape
    if len(shape) != 4 or shape[0] != B or shape[3] != hd or q.dtype is not bf16 or q.device != dev:
        raise ValueError(f"draft_attention: q must be bf16 [{B}, T, q_heads, {hd}] on {dev}, got {q.dtype} {list(shape)} on {q.device}")
    T, qh = shape[1], shape[2]
    if T > MAX_DRAFTS:
        raise ValueError(f"draft_attention: at most {MAX_DRAFTS} drafts per sequence, got {T}")
    if qh % H or qh == 0:
        raise ValueError(f"draft_attention: {qh} query heads are not a multiple of {H} KV heads")
    if out is None:
        # nodes behind counts are not written: zeros there rather than what the memory held
        out = (torch.empty if counts is None else torch.zeros)(B, T, qh, hd, dtype=bf16, device=dev)
    elif out.shape != shape or out.dtype is not bf16 or out.device != dev:
        raise ValueError("draft_attention: out must be like q")
    elif _overlap(out.stride(), B, T, qh * hd):
        raise ValueError("draft_attention: rows of out overlap")
    qs, os = q.stride(), out.stride()
    if qs[3] != 1 or os[3] != 1 or (qh > 1 and (qs[2] != hd or os[2] != hd)):
        raise ValueError("draft_attention: heads of q and out must be dense")
    if visible is not None and (visible.dtype is not torch.int64 or visible.shape != (B, T) or visible.device != dev or not visible.is_contiguous()):
        raise ValueError(f"draft_attention: visible must be a contiguous int64 [{B}, {T}] on {dev}")
    p, n = _ints(pos, "draft_attention: pos", dev, (B,)), _ints(counts, "draft_attention: counts", dev, (B,))
    args = (q.data_ptr(), out.data_ptr(), qs[0], qs[1], os[0] if B > 1 else 0, os[1] if T > 1 else 0, p, n, 0 if visible is None else visible.data_ptr(), T, qh, window, splits,
            hd ** -0.5 if scale is None else scale)
    key = (T, qh, window, splits, scale)
    floats = cache._scratch.get(key)
    if floats is None:                           # a function of the sizes alone; also checks the arguments
        with torch.cuda.device(cache._index):    # (-1: none) how the work is cut depends on the device
            floats = _lib().mesh_draft_attention_scratch(cache._at, _ARGS.pack(*args, 0, cache._status))
        if floats < 0:
            raise ValueError(_native.last_error())
        if len(cache._scratch) > 256:            # a scale of every call's own
            cache._scratch.clear()
        cache._scratch[key] = floats
    if B == 0 or T == 0:
        return out
    if floats == 0 or cache._index < 0:          # one kernel, whose clusters join their shares themselves
        _launch(cache._index, "mesh_draft_attention", 1, cache._at, _ARGS.pack(*args, 0, cache._status))
    else:
        # scratch of the call's own: calls on other streams and other captured graphs share nothing
        scratch = torch.empty(floats, dtype=torch.float32, device=dev)
        _launch(cache._index, "mesh_draft_attention", 2, cache._at, _ARGS.pack(*args, scratch.data_ptr(), cache._status))
    return out
