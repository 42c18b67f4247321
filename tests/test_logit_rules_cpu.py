"""LogitRules refuses what a step could not run with, before any step does."""
import pytest

torch = pytest.importorskip("torch")

import saccade_core as sc

MASK = torch.full((2, 4), -1, dtype=torch.int32)


@pytest.mark.parametrize("kw", [
    dict(mask=MASK.long()), dict(mask=MASK[0]), dict(mask=torch.full((4, 2), -1, dtype=torch.int32).T),
    dict(mask=MASK[:1]), dict(mask_row=[0, 0]), dict(mask=MASK, mask_row=[0]), dict(mask=MASK, mask_row=[0, 1, 1]),
    dict(mask=MASK, mask_row=[0, 2]), dict(mask=MASK[:0], mask_row=[-1, 0])], ids=str)
def test_masks_that_do_not_fit_are_refused(kw):
    with pytest.raises(ValueError, match="mask"):
        sc.LogitRules(2, "cpu", **kw)


def test_masks_that_fit():
    r = sc.LogitRules(2, "cpu", mask=MASK)
    assert r.mask is MASK and r.mask_row is None
    assert sc.LogitRules(2, "cpu", mask=MASK[:1], mask_row=[-1, 0]).mask_row.tolist() == [-1, 0]
    assert sc.LogitRules(2, "cpu", mask=MASK[:0], mask_row=[-1, -1]).mask.shape[0] == 0


def test_rules_of_another_batch_device_or_vocabulary_are_refused():
    cpu = torch.device("cpu")
    r = sc.LogitRules(2, "cpu", repetition=1.1, mask=MASK)
    r.check(2, cpu, 128)
    for args in ((3, cpu, 128), (1, cpu, 128), (2, torch.device("meta"), 128), (2, cpu, 129)):
        with pytest.raises(ValueError):
            r.check(*args)
    sc.LogitRules(2, "cpu").check(2, torch.device("meta"), 1 << 20)
