"""Constraints on logits: penalties for repeated tokens, biases, a grammar mask, and the token chosen from what is left.

Beside ``ops.decode.decode_argmax``, which chooses among the logits as they are.  Reference: vocabulary selection
(design/prepared-machine.md: "Vocabulary selection follows MAXLOC").
"""
from __future__ import annotations

import ctypes
from ctypes import c_int, c_longlong, c_void_p

import torch

from .. import _native
from .cache import _ints, _launch


class _Logits(ctypes.Structure):
    """``MeshLogits`` (csrc/ops/draft_api.h)."""
    _fields_ = [("logits", c_void_p), ("ldl", c_longlong), ("out", c_void_p), ("ldo", c_longlong), ("half", c_int),
                ("rows", c_int), ("vocab", c_int), ("vocab_offset", c_int),
                ("history", c_void_p), ("ldh", c_longlong), ("hist", c_int), ("history_len", c_void_p), ("prompt_len", c_void_p),
                ("repetition", c_void_p), ("presence", c_void_p), ("frequency", c_void_p),
                ("bias_ids", c_void_p), ("bias", c_void_p), ("ldb", c_longlong), ("nbias", c_int), ("bias_len", c_void_p),
                ("allowed", c_void_p), ("ldw", c_longlong), ("tokens", c_void_p)]


def _rows2d(t: torch.Tensor, name: str, dtype, device, rows: int, cols: int | None = None) -> torch.Tensor:
    """A matrix of ``rows`` rows whose last dimension is dense; a stride of 0 between rows (one list for all) is allowed."""
    if t.dim() != 2 or t.shape[0] != rows or (cols is not None and t.shape[1] != cols) or t.dtype != dtype or t.device != device:
        raise ValueError(f"constrain_logits: {name} must be {dtype} [{rows}, {'n' if cols is None else cols}] on {device}, "
                         f"got {t.dtype} {list(t.shape)} on {t.device}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"constrain_logits: rows of {name} must be dense")
    return t


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

    ``out``: where the result goes, in the logits' type (may be ``logits``); ``tokens [R]`` int32: the id of the largest result (not yet
    rounded to the logits' type), the lowest of equal ones, -1 where nothing is above -inf (NaN is never chosen).  At least one of them; returns
    ``out``, or ``tokens`` without it.  Lists may be shared by rows (``expand``).  With a vocabulary cut over ranks: ``out=logits`` on every
    rank, then ``decode_argmax``."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or not logits.is_cuda:
        raise ValueError(f"constrain_logits: logits must be fp32 or bf16 [R, V] on a GPU, got {logits.dtype} {list(logits.shape)} on {logits.device}")
    R, V = logits.shape
    dev = logits.device
    if V == 0 or (V > 1 and logits.stride(1) != 1):
        raise ValueError("constrain_logits: rows of the logits must be dense and not empty")
    if out is None and tokens is None:
        raise ValueError("constrain_logits: ask for out, for tokens, or for both")
    if R > 1 and logits.stride(0) < V:
        raise ValueError("constrain_logits: rows of the logits overlap")
    a = _Logits(logits=logits.data_ptr(), ldl=logits.stride(0), half=int(logits.dtype == torch.bfloat16), rows=R, vocab=V, vocab_offset=vocab_offset)
    if out is not None:
        _rows2d(out, "out", logits.dtype, dev, R, V)
        if R > 1 and out.stride(0) < V:
            raise ValueError("constrain_logits: rows of out overlap")
        a.out, a.ldo = out.data_ptr(), out.stride(0)
    if history is not None:
        _rows2d(history, "history", torch.int32, dev, R)
        if history.shape[1] > 65535:
            raise ValueError(f"constrain_logits: a history of at most 65535 tokens, got {history.shape[1]}")
        a.history, a.ldh, a.hist = history.data_ptr(), history.stride(0), history.shape[1]
    elif any(x is not None for x in (history_len, prompt_len, repetition, presence, frequency)):
        raise ValueError("constrain_logits: penalties need a history")
    a.history_len = _ints(history_len, "constrain_logits: history_len", dev, R)
    a.prompt_len = _ints(prompt_len, "constrain_logits: prompt_len", dev, R)
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None:
            if t.dtype != torch.float32 or t.shape != (R,) or t.device != dev or not t.is_contiguous():
                raise ValueError(f"constrain_logits: {name} must be contiguous fp32 [{R}] on {dev}")
            setattr(a, name, t.data_ptr())
    if (bias is None) != (bias_ids is None) or (bias is None and bias_len is not None):
        raise ValueError("constrain_logits: bias and bias_ids come together")
    if bias is not None:
        _rows2d(bias_ids, "bias_ids", torch.int32, dev, R)
        _rows2d(bias, "bias", torch.float32, dev, R, bias_ids.shape[1])
        if R > 1 and bias.stride(0) != bias_ids.stride(0):
            raise ValueError("constrain_logits: bias and bias_ids must have the same row stride")
        if bias.shape[1] > 32767:
            raise ValueError(f"constrain_logits: at most 32767 biases, got {bias.shape[1]}")
        a.bias_ids, a.bias, a.ldb, a.nbias = bias_ids.data_ptr(), bias.data_ptr(), bias.stride(0), bias.shape[1]
    a.bias_len = _ints(bias_len, "constrain_logits: bias_len", dev, R)
    if allowed is not None:
        _rows2d(allowed, "allowed", torch.int32, dev, R, (V + 31) // 32)
        a.allowed, a.ldw = allowed.data_ptr(), allowed.stride(0)
    a.tokens = _ints(tokens, "constrain_logits: tokens", dev, R)
    if R:
        _launch(dev, "mesh_constrain_logits", ctypes.byref(a))
        _native.count_launch()
    return out if out is not None else tokens
