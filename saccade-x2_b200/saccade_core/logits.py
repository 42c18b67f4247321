"""process_logits: penalties for repeated tokens, biases and grammar masks on a step's logits, with the
best token of each row (the argmax of saccade-runner/src/bin/verify.rs:98-130, which decodes without any
of them)."""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import LIB
from .op import _DT
from .paged import _call, _size, _status


def _vector(t: torch.Tensor, what: str, n: int, dtype: torch.dtype, dev: int) -> int:
    if t.dim() != 1 or t.shape[0] != n or t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor [{n}] on the logits' device")
    return t.data_ptr()


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
    dtype, dev = logits.dtype, logits.get_device()
    if logits.dim() != 2 or dtype not in _DT or dev < 0:
        raise ValueError("logits must be a float32, float16 or bfloat16 CUDA tensor [rows, vocab]")
    rows, vocab = logits.shape
    stride, one = logits.stride()
    if one != 1 and vocab > 1:
        raise ValueError("each row of the logits must be contiguous")
    if vocab < 1 or vocab_begin < 0:
        raise ValueError("the logits must have a token, and vocab_begin must not be negative")
    if out is None:
        out = logits.new_empty((rows, vocab))
        out_stride = vocab
    else:
        out_stride, one = out.stride() if out.dim() == 2 else (0, 0)
        if out.shape != logits.shape or out.dtype is not dtype or out.get_device() != dev or (one != 1 and vocab > 1):
            raise ValueError("out must be of the logits' shape, type and device, each row contiguous")
    i32, f32 = torch.int32, torch.float32
    width, p_hist, p_hlen, p_plen = 0, None, None, None
    if history is not None:
        if history.dim() != 2 or history.shape[0] != rows or history.dtype is not i32 or history.get_device() != dev \
                or not history.is_contiguous():
            raise ValueError(f"history must be a contiguous int32 tensor [{rows}, width] on the logits' device")
        if hist_len is None:
            raise ValueError("a history needs hist_len")
        width, p_hist = history.shape[1], history.data_ptr()
        p_hlen = _vector(hist_len, "hist_len", rows, i32, dev)
        if prompt_len is not None:
            p_plen = _vector(prompt_len, "prompt_len", rows, i32, dev)
    elif hist_len is not None or prompt_len is not None:
        raise ValueError("hist_len and prompt_len are a history's")
    p_rep = None if repetition is None else _vector(repetition, "repetition", rows, f32, dev)
    p_pres = None if presence is None else _vector(presence, "presence", rows, f32, dev)
    p_freq = None if frequency is None else _vector(frequency, "frequency", rows, f32, dev)
    nbias, p_bptr, p_bids, p_bvals = 0, None, None, None
    if bias_ptr is not None:
        if bias_ids is None or bias_vals is None or bias_ids.dim() != 1:
            raise ValueError("bias_ptr needs bias_ids and bias_vals [entries]")
        nbias = bias_ids.shape[0]
        p_bptr = _vector(bias_ptr, "bias_ptr", rows + 1, i32, dev)
        p_bids = _vector(bias_ids, "bias_ids", nbias, i32, dev)
        p_bvals = _vector(bias_vals, "bias_vals", nbias, f32, dev)
    elif bias_ids is not None or bias_vals is not None:
        raise ValueError("bias entries need bias_ptr")
    masks, words, p_mask, p_mrow = 0, 0, None, None
    if mask is not None:
        if mask.dim() != 2 or mask.dtype is not i32 or mask.get_device() != dev or not mask.is_contiguous():
            raise ValueError("mask must be a contiguous int32 tensor [masks, words] on the logits' device")
        masks, words = mask.shape
        if words * 32 < vocab_begin + vocab:
            raise ValueError(f"a mask of {words} words does not cover token {vocab_begin + vocab - 1}")
        if mask_row is not None:
            p_mrow = _vector(mask_row, "mask_row", rows, i32, dev)
        elif masks < rows:
            raise ValueError("fewer masks than rows (mask_row names each row's)")
        p_mask = mask.data_ptr()
    elif mask_row is not None:
        raise ValueError("mask_row needs a mask")
    best = value = scratch = None
    nbytes = 0
    if return_best:
        best = logits.new_empty(rows, dtype=torch.int64)
        value = logits.new_empty(rows)
        nbytes = _size(dev, "sc_qwen2_process_logits_scratch", rows, vocab)
        scratch = best.new_empty(nbytes // 8)
    if rows > 0:
        _call(dev, LIB.sc_qwen2_process_logits, logits.data_ptr(), _DT[dtype], rows, vocab, stride, vocab_begin, p_hist,
              width, p_plen, p_hlen, p_rep, p_pres, p_freq, p_bptr, p_bids, p_bvals, nbias, p_mask, words, masks, p_mrow,
              out.data_ptr(), out_stride, None if best is None else best.data_ptr(),
              None if value is None else value.data_ptr(), None if scratch is None else scratch.data_ptr(), nbytes,
              _status(status, dev))
    return (out, best, value) if return_best else out
