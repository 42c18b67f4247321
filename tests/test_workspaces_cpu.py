"""The linears' workspaces as ragged token counts grow them."""
import pytest

torch = pytest.importorskip("torch")

from saccade_core.op import _Workspaces


class Stream:
    cuda_stream = 1


def test_kept_workspaces_stay_within_a_multiple_of_the_largest_need():
    """A need that grows a little with every call: a replaced workspace is kept (graphs may hold it), so few may be
    replaced."""
    ws, dev = _Workspaces(), torch.device("cpu")
    need = 1 << 20
    for _ in range(300):
        need += 5000
        got = ws.get(dev, Stream, need)
        assert got.numel() >= need and not got.any()
        assert ws.get(dev, Stream, need // 2) is got
    kept = sum(t.numel() for t in ws._retired) + got.numel()
    assert len(ws._retired) <= 3 and kept <= 4.5 * need  # 1.5 x the need, and twice that before it
