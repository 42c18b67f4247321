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
