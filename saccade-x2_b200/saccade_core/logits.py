"""process_logits: penalties for repeated tokens, biases and grammar masks on a step's logits, with the
best token of each row (the argmax of saccade-runner/src/bin/verify.rs:98-130, which decodes without any
of them)."""
from __future__ import annotations

from typing import Optional

import torch

from .paged import _serve  # bound to the library there


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
    return _serve.process_logits(logits, history, prompt_len, hist_len, repetition, presence, frequency, bias_ptr, bias_ids,
                                 bias_vals, mask, mask_row, vocab_begin, out, return_best, status)
