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

from . import _lib
from ._lib import LIB, check
from .op import _DT


def _run_on(device: torch.device, call) -> None:
    """Runs `call(stream)` with the tensors' device current (kernels launch on the current one)."""
    if device.index == torch.cuda.current_device():
        check(call(torch.cuda.current_stream().cuda_stream))
    else:
        with torch.cuda.device(device):
            check(call(torch.cuda.current_stream().cuda_stream))


def _rows(t: torch.Tensor, what: str) -> int:
    """Row stride of a [tokens, heads, dim] tensor whose heads are contiguous."""
    if t.dim() != 3 or t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != t.shape[2]):
        raise ValueError(f"{what} must be [tokens, heads, head_dim] with each token's heads contiguous")
    return t.stride(0)


def _paged_args(k_pages, v_pages, block_table, cu_q, kv_len):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError("k_pages and v_pages must both be [pages, kv heads, page size, head dim] of one type")
    n, nkv, page, hd = k_pages.shape
    if k_pages.dtype not in _DT:
        raise ValueError("the cache must be float32, float16 or bfloat16")
    want = (page * hd, hd, 1)
    if k_pages.stride()[1:] != want or v_pages.stride()[1:] != want or k_pages.stride(0) != v_pages.stride(0):
        raise ValueError("each page must be contiguous, and k_pages and v_pages equally far apart")
    seqs = kv_len.shape[0] if kv_len.dim() == 1 else -1
    if (block_table.dtype != torch.int32 or cu_q.dtype != torch.int32 or kv_len.dtype != torch.int32 or
            block_table.dim() != 2 or block_table.shape[0] != seqs or cu_q.shape != (seqs + 1,)):
        raise ValueError("block_table [seqs, max pages], cu_q [seqs + 1] and kv_len [seqs] must be int32")
    if not (block_table.is_contiguous() and cu_q.is_contiguous() and kv_len.is_contiguous()):
        raise ValueError("block_table, cu_q and kv_len must be contiguous")
    dev = k_pages.device
    if dev.type != "cuda" or v_pages.device != dev or block_table.device != dev or cu_q.device != dev or kv_len.device != dev:
        raise ValueError("the pages, the block table and the lengths must be on one CUDA device")
    return n, nkv, page, hd, seqs, dev


def _status(status, dev):
    if status is None:
        return None
    if status.dtype != torch.int32 or status.device != dev or status.numel() < 1:
        raise ValueError("status must be an int32 tensor on the cache's device")
    return status.data_ptr()


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
    n, nkv, page, hd, seqs, dev = _paged_args(k_pages, v_pages, block_table, cu_q, kv_len)
    qs, ks, vs = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    tokens, nh = q.shape[0], q.shape[1]
    if q.shape[2] != hd or k.shape != (tokens, nkv, hd) or v.shape != k.shape:
        raise ValueError(f"q must be [tokens, heads, {hd}], k and v [tokens, {nkv}, {hd}]")
    if q.dtype not in _DT or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must be of one type")
    if (cos.dtype != torch.float32 or cos.dim() != 2 or cos.shape[1] != hd or cos.shape != sin.shape or
            sin.dtype != torch.float32 or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError(f"cos and sin must be contiguous float32 [positions, {hd}]")
    if q.device != dev or k.device != dev or v.device != dev or cos.device != dev or sin.device != dev:
        raise ValueError(f"every tensor must be on {dev}")
    if out is None:
        out = torch.empty((tokens, nh, hd), dtype=k_pages.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != k_pages.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {k_pages.dtype} tensor of q's shape on {dev}")
    if tokens == 0 or seqs == 0:
        return out
    st = _status(status, dev)
    _run_on(dev, lambda stream: LIB.sc_qwen2_paged_append(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _DT[q.dtype], qs, ks, vs, tokens, cos.data_ptr(), sin.data_ptr(),
        cos.shape[0], nh, nkv, hd, k_pages.data_ptr(), v_pages.data_ptr(), _DT[k_pages.dtype], n, k_pages.stride(0),
        page, block_table.data_ptr(), block_table.shape[1], cu_q.data_ptr(), kv_len.data_ptr(), seqs, out.data_ptr(),
        st, stream))
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
    n, nkv, page, hd, seqs, dev = _paged_args(k_pages, v_pages, block_table, cu_q, kv_len)
    qs = _rows(q, "q")
    tokens, nh = q.shape[0], q.shape[1]
    if q.shape[2] != hd or q.dtype != k_pages.dtype or q.device != dev:
        raise ValueError(f"q must be [tokens, heads, {hd}] {k_pages.dtype} on {dev}")
    if out is not None:
        out_dtype = out.dtype if out_dtype is None else out_dtype
        if out.shape != q.shape or out.dtype != out_dtype or out.device != dev or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {out_dtype} tensor of q's shape on {dev}")
    else:
        out_dtype = q.dtype if out_dtype is None else out_dtype
        out = torch.empty((tokens, nh, hd), dtype=out_dtype, device=dev)
    if out_dtype not in _DT:
        raise ValueError("out must be of the cache's type, or float16 from a float32 cache")
    lse = torch.empty((tokens, nh), dtype=torch.float32, device=dev) if return_lse else None
    if tokens > 0 and seqs > 0:
        max_q_len = min(int(max_q_len), tokens)
        nbytes = int(LIB.sc_qwen2_paged_attention_scratch(tokens, seqs, nh, nkv, hd, max_q_len, _DT[q.dtype]))
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        st = _status(status, dev)
        scale = hd ** -0.5 if scale is None else float(scale)
        _run_on(dev, lambda stream: LIB.sc_qwen2_paged_attention(
            q.data_ptr(), qs, k_pages.data_ptr(), v_pages.data_ptr(), _DT[q.dtype], n, k_pages.stride(0), page,
            block_table.data_ptr(), block_table.shape[1], cu_q.data_ptr(), kv_len.data_ptr(), seqs, tokens, nh, nkv, hd,
            max_q_len, int(max_kv_len), scale, out.data_ptr(), _DT[out_dtype], None if lse is None else lse.data_ptr(),
            None if scratch is None else scratch.data_ptr(), nbytes, st, stream))
    return (out, lse) if return_lse else out
