"""A paged KV cache: appending rotated keys and values, attention over the pages, and the pages' owner.

    paged_append      sc_qwen2_paged_append: rotates q and k, writes k and v into the pages
    paged_attention   sc_qwen2_paged_attention: causal attention of every sequence's new tokens
    PagePool          which pages are free (host side)
    PagedKVCache      a model's pages, its pool and the block tables of its sequences

The reference keeps one f32 cache tensor per sequence and concatenates to it (saccade-runner/src/
model.rs:228-236).  Here a cache of f32, f16 or bf16 is cut into pages [kv heads][page][head dim] that
sequences take as they grow; row b of the block table lists sequence b's pages in order.  Sequence b
owns the token rows cu_q[b]..cu_q[b + 1] and has kv_len[b] positions after them, so its i-th new token
sits at position kv_len[b] - q_len[b] + i.  Lengths and tables are device tensors: a captured graph
replays with new ones in the same tensors.  Calls run on the current stream of the tensors' device,
allocate nothing but their outputs and scratch (through torch's allocator) and do not synchronise.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional

import torch

from . import _serve
from ._lib import LIB, check
from .op import _DT


def _status_check(status: int) -> None:
    check(status)


_ENTRY_POINTS = ("sc_qwen2_paged_append", "sc_qwen2_paged_attention", "sc_qwen2_paged_attention_scratch",
                 "sc_qwen2_process_logits", "sc_qwen2_process_logits_scratch")
_serve.bind(_status_check, {n: ctypes.cast(getattr(LIB, n), ctypes.c_void_p).value for n in _ENTRY_POINTS})


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, cu_q: torch.Tensor,
                 kv_len: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates q and k by their positions' rows of cos / sin (f32 [positions, head_dim]), writes k and v
    into the pages and returns the rotated q [tokens, heads, head_dim] in the cache's type.
    q [tokens, heads, head_dim], k and v [tokens, kv heads, head_dim]: f32 or the cache's type, rows any
    distance apart (slices of one projection buffer).  out: where the rotated q goes (q itself works when
    it is contiguous and of the cache's type).  Rows behind the last sequence are left as they were, so
    with out=None their part of the result holds nothing.  status: int32 device word that a position or page
    outside the tables sets."""
    return _serve.paged_append(q, k, v, cos, sin, k_pages, v_pages, block_table, cu_q, kv_len, out, status)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    cu_q: torch.Tensor, kv_len: torch.Tensor, max_q_len: int, max_kv_len: int, *,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    out_dtype: Optional[torch.dtype] = None, return_lse: bool = False,
                    status: Optional[torch.Tensor] = None):
    """Causal attention of each sequence's new tokens over its cached positions (the new ones among them):
    out [tokens, heads, head_dim] = softmax(scale * q . k) v, and with return_lse also the f32
    [tokens, heads] log sum exp of the scores.  q [tokens, heads, head_dim] of the cache's type; scale
    1 / sqrt(head_dim) by default; out_dtype the cache's (or f16 from an f32 cache).  max_q_len and
    max_kv_len bound every sequence's new and cached lengths (they may be larger: a captured graph takes
    the capacity).  A token at a negative position attends nothing: 0, lse -inf.  Rows behind the last
    sequence are left as they were."""
    if out_dtype is None:
        code = -1
    elif out_dtype in _DT:
        code = _DT[out_dtype]
    else:
        raise ValueError("out must be of the cache's type, or float16 from a float32 cache")
    return _serve.paged_attention(q, k_pages, v_pages, block_table, cu_q, kv_len, max_q_len, max_kv_len, scale, out, code,
                                  return_lse, status)
