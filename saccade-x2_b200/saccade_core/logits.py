"""process_logits: penalties for repeated tokens, biases and grammar masks on a step's logits, with the
best token of each row (the argmax of saccade-runner/src/bin/verify.rs:98-130, which decodes without any
of them)."""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import LIB
from .op import _DT, _ptr
from .paged import _run_on, _status


def _vector(t: Optional[torch.Tensor], what: str, n: int, dtype: torch.dtype, dev: torch.device) -> None:
    if t is not None and (t.shape != (n,) or t.dtype != dtype or t.device != dev or not t.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous {dtype} tensor [{n}] on {dev}")


def process_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None,
                   prompt_len: Optional[torch.Tensor] = None, hist_len: Optional[torch.Tensor] = None,
                   repetition: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
                   frequency: Optional[torch.Tensor] = None, bias_ptr: Optional[torch.Tensor] = None,
                   bias_ids: Optional[torch.Tensor] = None, bias_vals: Optional[torch.Tensor] = None,
                   mask: Optional[torch.Tensor] = None, mask_row: Optional[torch.Tensor] = None, vocab_begin: int = 0,
                   out: Optional[torch.Tensor] = None, return_best: bool = False, status: Optional[torch.Tensor] = None):
    """Logits [rows, vocab] (f32, f16 or bf16) of the tokens vocab_begin..vocab_begin + vocab -> the processed
    logits (into `out`, which may be the logits themselves; a new tensor by default), with return_best also
    the largest one's id (int64 [rows], the first of equals) and value.  Per row and token, in f32:
      in the row's history:  x = x / repetition where x > 0, x * repetition elsewhere
      n times among its generated tokens:  x = x - frequency * n - (presence if n > 0)
      x = x + the token's (last) bias entry;  -inf where the row's mask does not allow the token
    history int32 [rows, width]: the first hist_len[r] ids are row r's, the first prompt_len[r] of them its
    prompt (no prompt_len: all generated); ids of other tokens than the slice's are passed over.
    repetition (> 0), presence, frequency: f32 [rows].  bias_ids / bias_vals entries bias_ptr[r]..bias_ptr[r + 1]
    (int32 [rows + 1]) are row r's, at most 4095 of them.  mask int32 [masks, words]: bit v % 32 of word
    v / 32 allows token v; mask_row int32 [rows] names each row's mask, negative for none (without it row r has
    mask r).  Ids are of the whole vocabulary throughout."""
    if logits.dim() != 2 or logits.dtype not in _DT or not logits.is_cuda:
        raise ValueError("logits must be a float32, float16 or bfloat16 CUDA tensor [rows, vocab]")
    rows, vocab = logits.shape
    dev = logits.device
    if logits.stride(1) != 1:
        raise ValueError("each row of the logits must be contiguous")
    if vocab < 1 or vocab_begin < 0:
        raise ValueError("the logits must have a token, and vocab_begin must not be negative")
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=dev)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev or out.stride(1) != 1:
        raise ValueError(f"out must be of the logits' shape and type on {dev}, its rows contiguous")
    width = 0
    if history is not None:
        if history.dim() != 2 or history.shape[0] != rows or history.dtype != torch.int32 or history.device != dev \
                or not history.is_contiguous():
            raise ValueError(f"history must be a contiguous int32 tensor [{rows}, width] on {dev}")
        if hist_len is None:
            raise ValueError("a history needs hist_len")
        width = history.shape[1]
    elif hist_len is not None or prompt_len is not None:
        raise ValueError("hist_len and prompt_len are a history's")
    _vector(hist_len, "hist_len", rows, torch.int32, dev)
    _vector(prompt_len, "prompt_len", rows, torch.int32, dev)
    for t, what in ((repetition, "repetition"), (presence, "presence"), (frequency, "frequency")):
        _vector(t, what, rows, torch.float32, dev)
    nbias = 0
    if bias_ptr is not None:
        if bias_ids is None or bias_vals is None or bias_ids.dim() != 1:
            raise ValueError("bias_ptr needs bias_ids and bias_vals [entries]")
        nbias = bias_ids.shape[0]
        _vector(bias_ptr, "bias_ptr", rows + 1, torch.int32, dev)
        _vector(bias_ids, "bias_ids", nbias, torch.int32, dev)
        _vector(bias_vals, "bias_vals", nbias, torch.float32, dev)
    elif bias_ids is not None or bias_vals is not None:
        raise ValueError("bias entries need bias_ptr")
    masks = words = 0
    if mask is not None:
        if mask.dim() != 2 or mask.dtype != torch.int32 or mask.device != dev or not mask.is_contiguous():
            raise ValueError(f"mask must be a contiguous int32 tensor [masks, words] on {dev}")
        masks, words = mask.shape
        if words * 32 < vocab_begin + vocab:
            raise ValueError(f"a mask of {words} words does not cover token {vocab_begin + vocab - 1}")
        if mask_row is None and masks < rows:
            raise ValueError("fewer masks than rows (mask_row names each row's)")
        if masks == 0:
            mask = None  # every mask_row is out of range: no row has one
    elif mask_row is not None:
        raise ValueError("mask_row needs a mask")
    _vector(mask_row, "mask_row", rows, torch.int32, dev)
    best = value = None
    if return_best:
        best = torch.empty(rows, dtype=torch.int64, device=dev)
        value = torch.empty(rows, dtype=logits.dtype, device=dev)
    if rows > 0:
        st = _status(status, dev)
        _run_on(dev, lambda stream: LIB.sc_qwen2_process_logits(
            logits.data_ptr(), _DT[logits.dtype], rows, vocab, logits.stride(0), vocab_begin, _ptr(history), width,
            _ptr(prompt_len), _ptr(hist_len), _ptr(repetition), _ptr(presence), _ptr(frequency), _ptr(bias_ptr),
            _ptr(bias_ids), _ptr(bias_vals), nbias, _ptr(mask), words, masks, _ptr(mask_row), out.data_ptr(),
            out.stride(0), _ptr(best), _ptr(value), st, stream))
    return (out, best, value) if return_best else out
