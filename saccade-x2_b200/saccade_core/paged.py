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

import functools
from typing import List, Optional

import torch

from ._lib import LIB, check
from .op import _DT


_raw_stream = torch._C._cuda_getCurrentRawStream  # the handle alone: a Stream object costs 3 us a call


def _call(dev: int, fn, *args) -> None:
    """check(fn(*args, current stream)) with device `dev` current (kernels launch on the current one)."""
    if dev == torch.cuda.current_device():
        st = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, _raw_stream(dev))
    if st:
        check(st)


def _rows(t: torch.Tensor, what: str) -> int:
    """Row stride of a [tokens, heads, dim] tensor whose heads are contiguous."""
    if t.dim() == 3:
        s0, s1, s2 = t.stride()
        if s2 == 1 and (s1 == t.shape[2] or t.shape[1] == 1):
            return s0
    raise ValueError(f"{what} must be [tokens, heads, head_dim] with each token's heads contiguous")


def _paged_args(k_pages, v_pages, block_table, cu_q, kv_len):
    """Checks a cache and its lengths: (pages, kv heads, page size, head dim, page stride, sequences, device)."""
    shape, dtype, strides = k_pages.shape, k_pages.dtype, k_pages.stride()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype is not dtype:
        raise ValueError("k_pages and v_pages must both be [pages, kv heads, page size, head dim] of one type")
    n, nkv, page, hd = shape
    if dtype not in _DT:
        raise ValueError("the cache must be float32, float16 or bfloat16")
    if strides[1:] != (page * hd, hd, 1) or v_pages.stride() != strides:
        raise ValueError("each page must be contiguous, and k_pages and v_pages equally far apart")
    i32, seqs = torch.int32, kv_len.shape[0] if kv_len.dim() == 1 else -1
    if (block_table.dtype is not i32 or cu_q.dtype is not i32 or kv_len.dtype is not i32 or block_table.dim() != 2 or
            block_table.shape[0] != seqs or cu_q.dim() != 1 or cu_q.shape[0] != seqs + 1):
        raise ValueError("block_table [seqs, max pages], cu_q [seqs + 1] and kv_len [seqs] must be int32")
    if not (block_table.is_contiguous() and cu_q.is_contiguous() and kv_len.is_contiguous()):
        raise ValueError("block_table, cu_q and kv_len must be contiguous")
    dev = k_pages.get_device()
    if not (dev >= 0 and dev == v_pages.get_device() == block_table.get_device() == cu_q.get_device() == kv_len.get_device()):
        raise ValueError("the pages, the block table and the lengths must be on one CUDA device")
    return n, nkv, page, hd, strides[0], seqs, dev


def _status(status: Optional[torch.Tensor], dev: int):
    if status is None:
        return None
    if status.dtype is not torch.int32 or status.get_device() != dev or status.numel() < 1:
        raise ValueError("status must be an int32 tensor on the other tensors' device")
    return status.data_ptr()


@functools.lru_cache(maxsize=4096)
def _size(dev: int, name: str, *sizes) -> int:
    """The answer of a scratch size function on device `dev`."""
    with torch.cuda.device(dev):
        return int(getattr(LIB, name)(*sizes))


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
    n, nkv, page, hd, stride, seqs, dev = _paged_args(k_pages, v_pages, block_table, cu_q, kv_len)
    qs, ks, vs = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    tokens, nh, qd = q.shape
    kshape, dtype, cdtype = k.shape, q.dtype, k_pages.dtype
    if qd != hd or kshape != (tokens, nkv, hd) or v.shape != kshape:
        raise ValueError(f"q must be [tokens, heads, {hd}], k and v [tokens, {nkv}, {hd}]")
    if (dtype is not torch.float32 and dtype is not cdtype) or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("q, k and v must all be float32 or all of the cache's type")
    tshape = cos.shape
    if (cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or len(tshape) != 2 or tshape[1] != hd or
            sin.shape != tshape or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError(f"cos and sin must be contiguous float32 [positions, {hd}]")
    if not dev == q.get_device() == k.get_device() == v.get_device() == cos.get_device() == sin.get_device():
        raise ValueError("every tensor must be on the cache's device")
    if out is None:
        out = k_pages.new_empty((tokens, nh, hd))
    elif out.shape != q.shape or out.dtype is not cdtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {cdtype} tensor of q's shape on the cache's device")
    if tokens == 0 or seqs == 0:
        return out
    _call(dev, LIB.sc_qwen2_paged_append, q.data_ptr(), k.data_ptr(), v.data_ptr(), _DT[dtype], qs, ks, vs, tokens,
          cos.data_ptr(), sin.data_ptr(), tshape[0], nh, nkv, hd, k_pages.data_ptr(), v_pages.data_ptr(), _DT[cdtype], n,
          stride, page, block_table.data_ptr(), block_table.shape[1], cu_q.data_ptr(), kv_len.data_ptr(), seqs,
          out.data_ptr(), _status(status, dev))
    return out


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
    n, nkv, page, hd, stride, seqs, dev = _paged_args(k_pages, v_pages, block_table, cu_q, kv_len)
    qs = _rows(q, "q")
    tokens, nh, qd = q.shape
    dtype = q.dtype
    if qd != hd or dtype is not k_pages.dtype or q.get_device() != dev:
        raise ValueError(f"q must be [tokens, heads, {hd}] {k_pages.dtype} on the cache's device")
    if out is not None:
        out_dtype = out.dtype if out_dtype is None else out_dtype
        if out.shape != q.shape or out.dtype is not out_dtype or out.get_device() != dev or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {out_dtype} tensor of q's shape on the cache's device")
    else:
        out_dtype = dtype if out_dtype is None else out_dtype
        out = q.new_empty((tokens, nh, hd), dtype=out_dtype)
    if out_dtype is not dtype and not (dtype is torch.float32 and out_dtype is torch.float16):
        raise ValueError("out must be of the cache's type, or float16 from a float32 cache")
    lse = q.new_empty((tokens, nh), dtype=torch.float32) if return_lse else None
    if tokens > 0 and seqs > 0:
        max_q_len = min(int(max_q_len), tokens)
        nbytes = _size(dev, "sc_qwen2_paged_attention_scratch", tokens, seqs, nh, nkv, hd, max_q_len, _DT[dtype])
        scratch = kv_len.new_empty((nbytes + 3) // 4)
        _call(dev, LIB.sc_qwen2_paged_attention, q.data_ptr(), qs, k_pages.data_ptr(), v_pages.data_ptr(), _DT[dtype], n,
              stride, page, block_table.data_ptr(), block_table.shape[1], cu_q.data_ptr(), kv_len.data_ptr(), seqs, tokens,
              nh, nkv, hd, max_q_len, int(max_kv_len), hd ** -0.5 if scale is None else scale, out.data_ptr(),
              _DT[out_dtype], None if lse is None else lse.data_ptr(), scratch.data_ptr(), nbytes, _status(status, dev))
    return (out, lse) if return_lse else out
