"""Constraints on logits: penalties for repeated tokens, biases, a grammar mask, and the token chosen from what is left.

Beside ``ops.decode.decode_argmax``, which chooses among the logits as they are.  Reference: vocabulary selection
(design/prepared-machine.md: "Vocabulary selection follows MAXLOC").
"""
from __future__ import annotations

import struct

import torch

from .cache import _index, _ints, _launch

# ``MeshLogits`` (csrc/ops/draft_api.h): logits, ldl, out, ldo, half, rows, vocab, vocab_offset, history, ldh, hist, history_len, prompt_len,
# repetition, presence, frequency, bias_ids, bias, ldb, nbias, bias_len, allowed, ldw, tokens
_ARGS = struct.Struct("@PqPqiiiiPqiPPPPPPPqiPPqP")


def _rows2d(t: torch.Tensor, name: str, dtype, device, rows: int, cols: int | None = None) -> tuple[int, int, int]:
    """(address, row stride, columns) of a matrix of ``rows`` rows whose last dimension is dense; a stride of 0 between rows (one
    list for all) is allowed."""
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows or (cols is not None and shape[1] != cols) or t.dtype is not dtype or t.device != device:
        raise ValueError(f"constrain_logits: {name} must be {dtype} [{rows}, {'n' if cols is None else cols}] on {device}, "
                         f"got {t.dtype} {list(shape)} on {t.device}")
    stride = t.stride()
    if stride[1] != 1 and shape[1] > 1:
        raise ValueError(f"constrain_logits: rows of {name} must be dense")
    return t.data_ptr(), stride[0], shape[1]


def _rows_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether rows of two matrices of one shape and type, at other places, may have bytes in common."""
    R, V = a.shape
    size, lda, ldb = a.element_size(), a.stride(0), b.stride(0)
    at, bt = a.data_ptr(), b.data_ptr()
    if R == 0 or at + ((R - 1) * lda + V) * size <= bt or bt + ((R - 1) * ldb + V) * size <= at:
        return False
    if R == 1:
        return at != bt
    return lda != ldb or not V * size <= (bt - at) % (lda * size) <= (lda - V) * size       # other columns of a wider matrix do not


def _per_row(t: torch.Tensor | None, name: str, device, rows: int) -> int:
    if t is None:
        return 0
    if t.dtype is not torch.float32 or t.shape != (rows,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"constrain_logits: {name} must be contiguous fp32 [{rows}] on {device}")
    return t.data_ptr()


def constrain_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None, history_len: torch.Tensor | None = None,
                     prompt_len: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                     presence: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                     bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None, bias_len: torch.Tensor | None = None,
                     allowed: torch.Tensor | None = None, vocab_offset: int = 0, out: torch.Tensor | None = None,
                     tokens: torch.Tensor | None = None) -> torch.Tensor:
    """``logits [R, V]`` fp32 or bf16 (rows dense; ids ``vocab_offset ..``), in this order, in fp32:

    * ``repetition [R]`` (> 0): ``l / r`` where ``l > 0``, else ``l * r``, for ids among the first ``history_len[r]`` of ``history [R, n]``;
    * ``frequency [R]``, ``presence [R]``: ``l - f * times - p`` for ids that stand ``times`` > 0 times in the history behind its
      first ``prompt_len[r]`` tokens;
    * ``bias [R, m]`` added at ``bias_ids [R, m]`` (the first ``bias_len[r]``); of an id listed twice the last entry counts;
    * ``allowed [R, ceil(V / 32)]`` int32: -inf where bit ``id % 32`` of word ``id // 32`` is clear (ids of this shard).

    ``out``: where the result goes, in the logits' type (may be ``logits``, but must not meet them otherwise); ``tokens [R]`` int32: the
    id of the largest result (not yet rounded to the logits' type), the lowest of equal ones, -1 where nothing is above -inf (NaN is never
    chosen).  At least one of them; returns ``out``, or ``tokens`` without it.  Lists may be shared by rows (``expand``).  With a vocabulary
    cut over ranks: ``out=logits`` on every rank, then ``decode_argmax``."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or not logits.is_cuda:
        raise ValueError(f"constrain_logits: logits must be fp32 or bf16 [R, V] on a GPU, got {logits.dtype} {list(logits.shape)} on {logits.device}")
    R, V = logits.shape
    dev = logits.device
    ldl, dense = logits.stride()
    if V == 0 or (V > 1 and dense != 1):
        raise ValueError("constrain_logits: rows of the logits must be dense and not empty")
    if out is None and tokens is None:
        raise ValueError("constrain_logits: ask for out, for tokens, or for both")
    if R > 1 and ldl < V:
        raise ValueError("constrain_logits: rows of the logits overlap")
    o, ldo = 0, 0
    if out is not None:
        o, ldo, _ = _rows2d(out, "out", logits.dtype, dev, R, V)
        if R > 1 and ldo < V:
            raise ValueError("constrain_logits: rows of out overlap")
        if (o != logits.data_ptr() or ldo != ldl) and _rows_meet(logits, out):
            raise ValueError("constrain_logits: out must be the logits themselves or memory apart from them")
    if not 0 <= vocab_offset <= 2**31 - 1 - V:
        raise ValueError(f"constrain_logits: ids {vocab_offset} .. {vocab_offset + V} are not all int32 and positive")
    h, ldh, hist = 0, 0, 0
    if history is not None:
        h, ldh, hist = _rows2d(history, "history", torch.int32, dev, R)
        if hist > 65535:
            raise ValueError(f"constrain_logits: a history of at most 65535 tokens, got {hist}")
    elif not (history_len is prompt_len is repetition is presence is frequency is None):
        raise ValueError("constrain_logits: penalties need a history")
    if (bias is None) != (bias_ids is None) or (bias is None and bias_len is not None):
        raise ValueError("constrain_logits: bias and bias_ids come together")
    ids, b, ldb, nbias = 0, 0, 0, 0
    if bias is not None:
        ids, ld_ids, nbias = _rows2d(bias_ids, "bias_ids", torch.int32, dev, R)
        b, ldb, _ = _rows2d(bias, "bias", torch.float32, dev, R, nbias)
        if R > 1 and ldb != ld_ids:
            raise ValueError("constrain_logits: bias and bias_ids must have the same row stride")
        if nbias > 32767:
            raise ValueError(f"constrain_logits: at most 32767 biases, got {nbias}")
    w, ldw = 0, 0
    if allowed is not None:
        w, ldw, _ = _rows2d(allowed, "allowed", torch.int32, dev, R, (V + 31) // 32)
    args = _ARGS.pack(logits.data_ptr(), ldl, o, ldo, logits.dtype is torch.bfloat16, R, V, vocab_offset, h, ldh, hist,
                      _ints(history_len, "constrain_logits: history_len", dev, (R,)), _ints(prompt_len, "constrain_logits: prompt_len", dev, (R,)),
                      _per_row(repetition, "repetition", dev, R), _per_row(presence, "presence", dev, R), _per_row(frequency, "frequency", dev, R),
                      ids, b, ldb, nbias, _ints(bias_len, "constrain_logits: bias_len", dev, (R,)), w, ldw,
                      _ints(tokens, "constrain_logits: tokens", dev, (R,)))
    if R:
        _launch(_index(dev), "mesh_constrain_logits", 1, args)
    return out if out is not None else tokens
