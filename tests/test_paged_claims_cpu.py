"""Who has the slots of a paged cache, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

import saccade_core as sc


class Decoder:
    pass


class Stream:
    waited = 0

    def synchronize(self):
        self.waited += 1


def cache():
    return sc.PagedKVCache(1, 10, 16, 1, 64, max_seqs=4, max_positions=160, device="cpu")


def test_a_dropped_decoders_pages_come_back_with_the_next():
    c, s = cache(), Stream()
    first = Decoder()
    c.claim(first, 3, s)
    for slot in range(3):
        c.reserve(slot, 20)
    c.reserve(3, 10)  # the user's own
    with pytest.raises(RuntimeError, match="another decoder"):
        c.claim(Decoder(), 1, s)
    assert c.free_pages == 3 and s.waited == 0
    del first
    second = Decoder()
    c.claim(second, 1, s)
    assert c.free_pages == 9 and s.waited == 1 and [len(c.pages(i)) for i in range(4)] == [0, 0, 0, 1]
    c.reserve(0, 33)
    c.claim(second, 1, s)  # again: keeps what it has
    assert c.free_pages == 6 and len(c.pages(0)) == 3
    c.give_back(Decoder())
    assert c.free_pages == 6
    c.give_back(second)
    c.give_back(second)
    assert c.free_pages == 9 and c.decoder() is None and len(c.pages(3)) == 1


def test_a_dropped_decoders_pages_come_back_when_pages_run_short():
    c, s = cache(), Stream()
    d = Decoder()
    c.claim(d, 2, s)
    c.reserve(0, 64)
    c.reserve(1, 64)
    with pytest.raises(RuntimeError, match="3 pages wanted, 2 of 10 free"):
        c.reserve(2, 48)
    assert len(c.pages(0)) == 4 and s.waited == 0
    del d
    c.reserve(3, 16)  # enough without them
    assert len(c.pages(0)) == 4 and s.waited == 0
    c.reserve(2, 48)
    assert c.free_pages == 6 and c.pages(0) == c.pages(1) == [] and s.waited == 1


def test_a_slot_taken_after_its_decoder_is_gone_stays_its_users():
    c = cache()
    d = Decoder()
    c.claim(d, 3, None)
    c.reserve(2, 20)
    del d
    c.release(2)
    c.reserve(2, 40)
    other = Decoder()
    c.claim(other, 1, None)
    assert len(c.pages(2)) == 3


def test_a_claimed_slot_that_is_released_by_hand_is_still_given_back():
    c, d = cache(), Decoder()
    c.claim(d, 2, None)
    c.reserve(0, 20)
    c.release(0)
    c.reserve(0, 20)
    c.reserve(1, 20)
    c.give_back(d)
    assert c.free_pages == 10


def test_a_dropped_decoders_slot_that_is_reserved_on_is_kept():
    """The slot is its user's from then on, with the pages that it has, also where pages run short."""
    c, d = cache(), Decoder()
    c.claim(d, 3, None)
    for slot in range(3):
        c.reserve(slot, 48)
    before = c.pages(0)
    del d
    c.reserve(0, 80)  # two more than its three, of one free: those of the other slots come back
    assert c.pages(0)[:3] == before and len(set(c.pages(0))) == 5 and c.block_table[0, :5].tolist() == c.pages(0)
    assert c.free_pages == 5 and c.pages(1) == c.pages(2) == []
    c.claim(Decoder(), 2, None)
    assert len(c.pages(0)) == 5
    c.release(0)
    assert c.free_pages == 10
