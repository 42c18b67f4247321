"""process_logits with lengths, ranges and mask rows out of range: what is cut, row by row, and the other rows as ever."""
import pytest

torch = pytest.importorskip("torch")

from test_logits_gpu import make, sc  # noqa: F401 - fixture

pytestmark = pytest.mark.gpu

ROW = 2


def alone(sc, x, kw, row, **put):  # noqa: F811
    """Row `row` by itself, with `put` as its values; bias=(first, end) as its entries."""
    one = lambda t: t[row:row + 1].contiguous()  # noqa: E731
    t = {k: one(kw[k]).clone() for k in ("history", "hist_len", "prompt_len", "repetition", "presence", "frequency", "mask_row")}
    for k, v in put.items():
        if k != "bias":
            t[k][0] = v
    ends = put.get("bias") or kw["bias_ptr"][row:row + 2].tolist()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = sc.process_logits(x[row:row + 1], mask=kw["mask"], bias_ids=kw["bias_ids"], bias_vals=kw["bias_vals"],
                            bias_ptr=torch.tensor(ends, dtype=torch.int32, device="cuda"), status=status, **t)
    assert int(status.item()) == 0
    return out[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("name,value", [
    ("hist_len", 101), ("hist_len", 2**31 - 1), ("hist_len", -1), ("prompt_len", 101), ("prompt_len", -7), ("mask_row", 2),
    ("mask_row", 2**31 - 1), ("bias_ptr", -1), ("bias_ptr", 2**31 - 1)])
def test_rows_out_of_range_are_cut_to_what_there_is(sc, dtype, name, value):  # noqa: F811
    x, kw = make(4, 3001, 0, 100, 20, 2, dtype, seed=6)
    kw["hist_len"][ROW], kw["prompt_len"][ROW] = 60, 20
    kw["mask_row"][ROW] = 1
    kw["bias_ptr"] = torch.tensor([0, 9, 21, 30, 44], dtype=torch.int32, device="cuda")
    kw["bias_ids"] = (torch.arange(50, device="cuda") * 37 % 61).to(torch.int32)
    kw["bias_vals"] = torch.randn(50, device="cuda")
    good = sc.process_logits(x, **kw)
    want = [good[r] for r in range(4)]
    if name == "hist_len":
        want[ROW] = alone(sc, x, kw, ROW, hist_len=min(max(value, 0), 100), prompt_len=0 if value < 0 else 20)
    elif name == "prompt_len":
        want[ROW] = alone(sc, x, kw, ROW, prompt_len=min(max(value, 0), 60))
    elif name == "mask_row":
        want[ROW] = alone(sc, x, kw, ROW, mask_row=-1)
    elif value < 0:  # the row before ends before it begins: no entries; this one begins at the first
        want[ROW - 1], want[ROW] = alone(sc, x, kw, ROW - 1, bias=(0, 0)), alone(sc, x, kw, ROW, bias=(0, 30))
    else:            # the row before has all that there are; this one begins behind them
        want[ROW - 1], want[ROW] = alone(sc, x, kw, ROW - 1, bias=(9, 50)), alone(sc, x, kw, ROW, bias=(0, 0))
    bad = dict(kw, **{name: kw[name].clone()})
    bad[name][ROW] = value
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = sc.process_logits(x, status=status, **bad)
    assert int(status.item()) != 0
    for r in range(4):
        assert torch.equal(out[r], want[r]), r
    assert not torch.equal(out[ROW], good[ROW]) or name == "prompt_len" or value == -1


def test_the_first_4095_bias_entries_of_a_row_apply(sc):  # noqa: F811
    x = torch.randn(2, 6000, device="cuda")
    ids = torch.arange(5000, dtype=torch.int32, device="cuda") + 7
    vals = torch.randn(5000, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = sc.process_logits(x, bias_ptr=torch.tensor([0, 5000, 5000], dtype=torch.int32, device="cuda"), bias_ids=ids,
                            bias_vals=vals, status=status)
    assert int(status.item()) != 0
    want = x.clone()
    want[0, 7:7 + 4095] += vals[:4095]
    assert torch.equal(out, want)
    status.zero_()
    out = sc.process_logits(x, bias_ptr=torch.tensor([0, 4095, 5000], dtype=torch.int32, device="cuda"), bias_ids=ids,
                            bias_vals=vals, status=status)
    assert int(status.item()) == 0
    want[1, 7 + 4095:7 + 5000] += vals[4095:]
    assert torch.equal(out, want)
