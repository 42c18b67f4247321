"""Logits processing:

    process_logits   sc_qwen2_process_logits on tensors
    LogitRules       the penalties, biases and masks of a batch of sequences, on the device

Penalties for repeated tokens, biases and grammar masks on a step's logits, with the
best token of each row (the argmax of saccade-runner/src/bin/verify.rs:98-130, which decodes without any
of them)."""
from __future__ import annotations

from typing import Dict, Optional, Sequence, Union

import torch

from .paged import _serve  # bound to the library there, or missing

MAX_HISTORY = 524287  # ids of a row's history (sc_qwen2_process_logits)


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
    history int32 [rows, width <= MAX_HISTORY]: the first hist_len[r] ids are row r's, the first prompt_len[r] of
    them its prompt (no prompt_len: all generated); ids of other tokens than the slice's are passed over.
    repetition (> 0), presence, frequency: f32 [rows].  bias_ids / bias_vals entries bias_ptr[r]..bias_ptr[r + 1]
    (int32 [rows + 1]) are row r's, at most 4095 of them.  mask int32 [masks, words]: bit v % 32 of word
    v / 32 allows token v; mask_row int32 [rows] names each row's mask, negative for none (without it row r has
    mask r).  Ids are of the whole vocabulary throughout."""
    return _serve.process_logits(logits, history, prompt_len, hist_len, repetition, presence, frequency, bias_ptr, bias_ids,
                                 bias_vals, mask, mask_row, vocab_begin, out, return_best, status)


class LogitRules:
    """What a batch's logits go through: repetition, presence and frequency penalties (a number, or one per
    sequence), bias (one {token: value} per sequence) and grammar masks (int32 [masks, words], one bit per
    token; mask_row: each sequence's mask or -1).  The tensors stay where they are, so a captured step follows
    what is written into them (a grammar's next mask, another penalty).  The rules are of `batch` sequences."""

    def __init__(self, batch: int, device, *, repetition: Union[None, float, Sequence[float]] = None,
                 presence: Union[None, float, Sequence[float]] = None,
                 frequency: Union[None, float, Sequence[float]] = None, bias: Optional[Sequence[Dict[int, float]]] = None,
                 mask: Optional[torch.Tensor] = None, mask_row: Optional[Sequence[int]] = None):
        self.batch = batch

        def floats(v, what):
            if v is None:
                return None
            t = torch.as_tensor(v, dtype=torch.float32)
            if t.dim() == 0:
                t = t.repeat(batch)
            if t.shape != (batch,):
                raise ValueError(f"{what} must be a number or one per sequence")
            return t.to(device)

        self.repetition = floats(repetition, "repetition")
        if self.repetition is not None and not bool((self.repetition > 0).all()):
            raise ValueError("a repetition penalty must be above 0")
        self.presence, self.frequency = floats(presence, "presence"), floats(frequency, "frequency")
        self.bias_ptr = self.bias_ids = self.bias_vals = None
        if bias is not None:
            if len(bias) != batch or max(map(len, bias), default=0) > 4095:
                raise ValueError("bias must be one {token: value} per sequence, of at most 4095 tokens each")
            ptr = [0]
            for b in bias:
                ptr.append(ptr[-1] + len(b))
            self.bias_ptr = torch.tensor(ptr, dtype=torch.int32, device=device)
            self.bias_ids = torch.tensor([t for b in bias for t in b], dtype=torch.int32, device=device)
            self.bias_vals = torch.tensor([x for b in bias for x in b.values()], dtype=torch.float32, device=device)
        if mask is not None and (mask.dim() != 2 or mask.dtype != torch.int32 or not mask.is_contiguous()):
            raise ValueError("mask must be a contiguous int32 tensor [masks, words]")
        if mask_row is None:
            if mask is not None and mask.shape[0] < batch:
                raise ValueError(f"{mask.shape[0]} masks for {batch} sequences (mask_row names each one's)")
        else:
            mask_row = list(mask_row)
            if mask is None or len(mask_row) != batch or max(mask_row, default=-1) >= mask.shape[0]:
                raise ValueError("mask_row must be each sequence's mask, one of those of `mask`, or -1")
        self.mask = None if mask is None else mask.to(device)
        self.mask_row = None if mask_row is None else torch.tensor(mask_row, dtype=torch.int32, device=device)

    def check(self, batch: int, device: torch.device, vocab: int) -> None:
        """ValueError where these rules are not of `batch` sequences over a vocabulary of `vocab` tokens on `device`."""
        if self.batch != batch:
            raise ValueError(f"rules of {self.batch} sequences for {batch}")
        tensors = (self.repetition, self.presence, self.frequency, self.bias_ptr, self.mask, self.mask_row)
        if any(t is not None and t.device != device for t in tensors):
            raise ValueError(f"the rules must be on {device}")
        if self.mask is not None and self.mask.shape[1] * 32 < vocab:
            raise ValueError(f"masks of {self.mask.shape[1]} words do not cover {vocab} tokens")

    def apply(self, logits: torch.Tensor, *, rows: Optional[torch.Tensor] = None, history=None, prompt_len=None,
              hist_len=None, vocab_begin: int = 0, out: Optional[torch.Tensor] = None,
              status: Optional[torch.Tensor] = None):
        """process_logits with these rules for all sequences, or for those of `rows` (a tensor of indices):
        (logits, best ids, best values)."""
        if rows is None:
            pick = lambda t: t  # noqa: E731
            bias = (self.bias_ptr, self.bias_ids, self.bias_vals)
            mask_row = self.mask_row
        else:
            pick = lambda t: None if t is None else t[rows].contiguous()  # noqa: E731
            bias, mask_row = self._bias_of(rows), pick(self.mask_row)
            if self.mask is not None and mask_row is None:
                mask_row = rows.to(device=self.mask.device, dtype=torch.int32)
        return process_logits(logits, history=history, prompt_len=prompt_len, hist_len=hist_len,
                              repetition=pick(self.repetition), presence=pick(self.presence),
                              frequency=pick(self.frequency), bias_ptr=bias[0], bias_ids=bias[1], bias_vals=bias[2],
                              mask=self.mask, mask_row=mask_row, vocab_begin=vocab_begin, out=out, return_best=True,
                              status=status)

    def _bias_of(self, rows: torch.Tensor):
        """The bias entries of some sequences as a list of their own."""
        if self.bias_ptr is None:
            return None, None, None
        ptr, idx = self.bias_ptr.tolist(), rows.tolist()
        keep = [e for r in idx for e in range(ptr[r], ptr[r + 1])]
        new = [0]
        for r in idx:
            new.append(new[-1] + ptr[r + 1] - ptr[r])
        dev = self.bias_ids.device
        take = torch.tensor(keep, dtype=torch.int64, device=dev)
        return torch.tensor(new, dtype=torch.int32, device=dev), self.bias_ids[take], self.bias_vals[take]
