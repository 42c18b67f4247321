"""A paged KV cache: appending rotated keys and values, attention over the pages, and the pages' owner.

    paged_append      sc_qwen2_paged_append: rotates q and k, writes k and v into the pages
    paged_attention   sc_qwen2_paged_attention: causal attention of every sequence's new tokens
    PagedKVCache      a model's pages of every layer, the free ones, and the block tables of its sequences

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
import weakref
from typing import List, Optional, Set

import torch

from ._lib import LIB, SC_EDEVICE, SC_ETIMEOUT, CTarqError, check
from .op import _DT


def _status_check(status: int) -> None:
    check(status)


_ENTRY_POINTS = ("sc_qwen2_paged_append", "sc_qwen2_paged_attention", "sc_qwen2_paged_attention_scratch",
                 "sc_qwen2_process_logits", "sc_qwen2_process_logits_scratch")


class _Missing:
    """In the module's place where it is not built or does not load: the rest of the package works without it."""

    def __init__(self, why: ImportError):
        self._why = why

    def __getattr__(self, name):
        raise ImportError(f"saccade_core._serve.{name}: the serving operators' module is missing (make -C csrc builds it)"
                          ) from self._why


try:
    from . import _serve
    _serve.bind(_status_check, {n: ctypes.cast(getattr(LIB, n), ctypes.c_void_p).value for n in _ENTRY_POINTS})
except ImportError as why:
    _serve = _Missing(why)


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, cu_q: torch.Tensor,
                 kv_len: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates q and k by their positions' rows of cos / sin (f32 [positions, head_dim]), writes k and v
    into the pages and returns the rotated q [tokens, heads, head_dim] in the cache's type.
    q [tokens, heads, head_dim], k and v [tokens, kv heads, head_dim]: f32 or the cache's type, rows any
    distance apart (slices of one projection buffer).  out: where the rotated q goes (q itself works when
    it is contiguous and of the cache's type; it must not lie over q, k or v otherwise).  Rows behind the last
    sequence are left as they were, so with out=None their part of the result holds nothing.  status: int32 device
    word that a position or page outside the tables sets."""
    return _serve.paged_append(q, k, v, cos, sin, k_pages, v_pages, block_table, cu_q, kv_len, out, status)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    cu_q: torch.Tensor, kv_len: torch.Tensor, max_q_len: int, max_kv_len: int, *,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    out_dtype: Optional[torch.dtype] = None, return_lse: bool = False,
                    status: Optional[torch.Tensor] = None):
    """Causal attention of each sequence's new tokens over its cached positions (the new ones among them):
    out [tokens, heads, head_dim] = softmax(scale * q . k) v, and with return_lse also the f32
    [tokens, heads] log sum exp of the scores.  q [tokens, heads, head_dim] of the cache's type; scale
    1 / sqrt(head_dim) by default; out_dtype the cache's (or f16 from an f32 cache).  out may be a contiguous
    q.  max_q_len and max_kv_len bound every sequence's new and cached lengths (they may be larger: a captured
    graph takes the capacity).  A token at a negative position attends nothing: 0, lse -inf.  Rows behind the
    last sequence are left as they were."""
    if out_dtype is None:
        code = -1
    elif out_dtype in _DT:
        code = _DT[out_dtype]
    else:
        raise ValueError("out must be of the cache's type, or float16 from a float32 cache")
    return _serve.paged_attention(q, k_pages, v_pages, block_table, cu_q, kv_len, max_q_len, max_kv_len, scale, out, code,
                                  return_lse, status)


class PagedKVCache:
    """Every layer's pages of a model, which of them are free, and the pages of up to max_seqs sequences.

    k[layer], v[layer]: [pages, kv heads, page size, head dim]; a sequence (slot) has the same page
    numbers in every layer.  block_table [max_seqs, pages of max_positions] and kv_len [max_seqs] live on
    the device.  reserve() and release() run on the host and write the slot's row of the block table
    on the current stream; the steps that read it are ordered behind them."""

    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, *, max_seqs: int,
                 max_positions: int, dtype: torch.dtype = torch.float16, device="cuda:0"):
        if layers < 1 or num_pages < 1 or kv_heads < 1 or max_seqs < 1 or max_positions < 1:
            raise ValueError("a cache needs layers, pages, KV heads, sequences and positions")
        if page_size < 8 or page_size > 256 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two in 8..256")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if dtype not in _DT:
            raise ValueError("the cache must be float32, float16 or bfloat16")
        self.page_size, self.num_pages, self.dtype = page_size, num_pages, dtype
        self.max_seqs, self.max_positions, self.device = max_seqs, max_positions, torch.device(device)
        shape = (num_pages, kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layers)]
        self.block_table = torch.zeros(max_seqs, -(-max_positions // page_size), dtype=torch.int32, device=self.device)
        self.kv_len = torch.zeros(max_seqs, dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(max_seqs)]
        self.decoder = lambda: None  # a reference to the decoder that runs on the slots
        self._claimed: Set[int] = set()  # the slots it has, and its stream
        self._claimed_stream = None

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages(self, slot: int) -> List[int]:
        """The slot's pages, in order."""
        return list(self._pages[self._slot(slot)])

    def _slot(self, slot: int) -> int:
        if not 0 <= slot < self.max_seqs:
            raise ValueError(f"slot {slot}: the cache has {self.max_seqs}")
        return slot

    def reserve(self, slot: int, positions: int) -> None:
        """Gives the slot the pages that `positions` positions need (it keeps those it has); RuntimeError, and
        nothing changed, where not enough are free."""
        if positions < 0 or positions > self.max_positions:
            raise ValueError(f"{positions} positions: the cache is made for up to {self.max_positions}")
        have = self._pages[self._slot(slot)]
        if self.decoder() is None:
            self._claimed.discard(slot)  # of a decoder that is gone: it is kept, for this caller
        need = -(-positions // self.page_size) - len(have)
        if need <= 0:
            return
        if need > len(self._free):
            self._reclaim()
        if need > len(self._free):
            raise RuntimeError(f"{need} pages wanted, {len(self._free)} of {self.num_pages} free")
        new = [self._free.pop() for _ in range(need)]
        row = torch.tensor(new, dtype=torch.int32).pin_memory() if self.device.type == "cuda" else torch.tensor(
            new, dtype=torch.int32)
        self.block_table[slot, len(have):len(have) + need].copy_(row, non_blocking=True)
        have.extend(new)

    def release(self, slot: int) -> None:
        """Takes the slot's pages back (what they hold stays until another sequence writes them)."""
        self._free.extend(reversed(self._pages[self._slot(slot)]))
        self._pages[slot] = []
        self.kv_len[slot] = 0
        if self.decoder() is None:
            self._claimed.discard(slot)

    def claim(self, decoder, slots: int, stream) -> None:
        """Slots 0 .. slots - 1 are `decoder`'s, which works on `stream`, until give_back(); RuntimeError where another
        decoder has not given its slots back.  Those of one that is gone are released first."""
        if self.decoder() not in (None, decoder):
            raise RuntimeError("another decoder runs on this cache; its finish() gives the sequences back")
        self._reclaim()
        self.decoder, self._claimed, self._claimed_stream = weakref.ref(decoder), set(range(slots)), stream

    def give_back(self, decoder) -> None:
        """Releases the slots that `decoder` has claimed (its work on them has ended), if it has any."""
        if self.decoder() is decoder:
            self.decoder = lambda: None
            for slot in sorted(self._claimed):
                self.release(slot)

    def _reclaim(self) -> None:
        """Releases what a decoder has claimed that is gone without giving it back, after its last steps."""
        if self._claimed and self.decoder() is None:
            if self._claimed_stream is not None:
                self._claimed_stream.synchronize()
            for slot in sorted(self._claimed):
                self.release(slot)

    def check_device(self) -> None:
        """Raises where a kernel met a position, page or length outside the tables (or a wait ran out)."""
        st = int(self.status.item())
        if st:
            self.status.zero_()
            raise CTarqError(SC_ETIMEOUT if st == 1 else SC_EDEVICE,
                             "a wait ran out in a paged-cache kernel" if st == 1 else
                             "a position, page or length outside the paged cache's tables")
