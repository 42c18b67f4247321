"""What PagedDecoder refuses before it touches a device."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

import saccade_core as sc
from saccade_core import qwen2 as q2


def test_a_history_wider_than_the_logits_take():
    """max_positions tokens and the one that the last of them gives."""
    for positions in (524287, 1 << 20):
        cache = sc.PagedKVCache(1, 1, 8, 1, 64, max_seqs=1, max_positions=positions, device="cpu")
        with pytest.raises(ValueError, match="history"):
            q2.PagedDecoder(SimpleNamespace(cache=cache, device=torch.device("cpu")), 1)


def test_a_cache_without_heads():
    with pytest.raises(ValueError, match="KV heads"):
        sc.PagedKVCache(1, 4, 16, 0, 64, max_seqs=1, max_positions=8, device="cpu")


def test_generating_nothing():
    """Refused before the prompts run: there is no token to return."""
    dec = q2.PagedDecoder.__new__(q2.PagedDecoder)
    for steps in (0, -1):
        with pytest.raises(ValueError, match="steps"):
            dec.generate([torch.zeros(3, dtype=torch.int64)], steps)
