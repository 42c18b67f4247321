"""The serving operators' refusals and bookkeeping, without a GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import saccade_core as sc
from saccade_core import _lib


def test_tensors_off_the_gpu_are_refused():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    q, kv = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, 2, 64, dtype=torch.float16)
    t = torch.zeros(8, 64)
    with pytest.raises(ValueError, match="one CUDA device"):
        sc.paged_append(q, kv, kv, t, t, k, k, i(1, 4), i(2), i(1))
    with pytest.raises(ValueError, match="one CUDA device"):
        sc.paged_attention(q, k, k, i(1, 4), i(2), i(1), 3, 64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        sc.process_logits(torch.zeros(2, 9))


@pytest.mark.parametrize("what,kw", [
    ("of one type", dict(v=torch.zeros(4, 2, 16, 64))),
    ("of one type", dict(v=torch.zeros(4, 2, 16, 32, dtype=torch.float16))),
    ("contiguous", dict(k=torch.zeros(4, 16, 2, 64, dtype=torch.float16).transpose(1, 2),
                        v=torch.zeros(4, 16, 2, 64, dtype=torch.float16).transpose(1, 2))),
    ("float32, float16 or bfloat16", dict(k=torch.zeros(4, 2, 16, 64, dtype=torch.float64),
                                          v=torch.zeros(4, 2, 16, 64, dtype=torch.float64))),
    ("must be int32", dict(table=torch.zeros(1, 4, dtype=torch.int64))),
    ("must be int32", dict(cu=torch.zeros(1, dtype=torch.int32))),
    ("must be int32", dict(kv=torch.zeros(1, 1, dtype=torch.int32))),
    ("must be a tensor", dict(table=[1, 2])),
])
def test_caches_of_another_shape_are_refused(what, kw):
    a = dict(k=torch.zeros(4, 2, 16, 64, dtype=torch.float16), v=torch.zeros(4, 2, 16, 64, dtype=torch.float16),
             table=torch.zeros(1, 4, dtype=torch.int32), cu=torch.zeros(2, dtype=torch.int32),
             kv=torch.zeros(1, dtype=torch.int32)) | kw
    with pytest.raises(ValueError, match=what):
        sc.paged_attention(torch.zeros(3, 4, 64, dtype=torch.float16), a["k"], a["v"], a["table"], a["cu"], a["kv"], 1, 1)


def _buf(n=1 << 16):
    raw = ctypes.create_string_buffer(n + 256)
    at = (ctypes.addressof(raw) + 255) & ~255
    return raw, at


class Call:
    """The C entry points' arguments as a call with nothing wrong has them, but for `tokens` = 0: a call that passes
    every check then returns SC_OK without touching a device."""

    def __init__(self):
        self.keep, self.p = _buf()

    def append(self, **kw):
        p = self.p
        a = dict(q=p, k=p, v=p, in_dtype=_lib.SC_F32, qs=256, ks=128, vs=128, tokens=4, cos=p, sin=p, max_pos=64, nh=4,
                 nkv=2, hd=64, kp=p, vp=p, dtype=_lib.SC_F16, pages=4, stride=2 * 16 * 64, page=16, table=p, max_pages=4,
                 cu=p, kv=p, seqs=1, out=p, status=None, stream=None) | kw
        return _lib.LIB.sc_qwen2_paged_append(*a.values())

    def attention(self, **kw):
        p = self.p
        a = dict(q=p, qs=256, kp=p, vp=p, dtype=_lib.SC_F16, pages=4, stride=2 * 16 * 64, page=16, table=p, max_pages=4,
                 cu=p, kv=p, seqs=1, tokens=4, nh=4, nkv=2, hd=64, max_q=1, max_kv=1 << 20, scale=0.125, out=p,
                 out_dtype=_lib.SC_F16, lse=None, scratch=p, nbytes=1 << 40, status=None, stream=None) | kw
        return _lib.LIB.sc_qwen2_paged_attention(*a.values())

    def logits(self, **kw):
        p = self.p
        a = dict(x=p, dtype=_lib.SC_F32, rows=2, vocab=100, stride=100, begin=0, hist=None, width=0, plen=None, hlen=None,
                 rep=None, pres=None, freq=None, bptr=None, bids=None, bvals=None, nbias=0, mask=None, words=0, masks=0,
                 mrow=None, out=p, out_stride=100, best=None, value=None, scratch=None, nbytes=0, status=None,
                 stream=None) | kw
        return _lib.LIB.sc_qwen2_process_logits(*a.values())


CACHE = [dict(dtype=3), dict(kp=None), dict(vp=None), dict(table=None), dict(cu=None), dict(kv=None), dict(hd=32),
         dict(hd=96), dict(hd=256), dict(nkv=0), dict(nh=0), dict(nh=3), dict(nh=132), dict(page=4), dict(page=512),
         dict(page=24), dict(pages=0), dict(stride=2 * 16 * 64 - 1), dict(max_pages=0), dict(max_pages=1 << 28),
         dict(seqs=0), dict(seqs=1 << 21), dict(tokens=1 << 30), dict(tokens=-1)]


@pytest.mark.parametrize("kw", CACHE + [
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cos=None), dict(sin=None), dict(in_dtype=_lib.SC_BF16),
    dict(max_pos=0), dict(qs=255), dict(ks=127), dict(vs=127)], ids=str)
def test_append_refuses(kw):
    c = Call()
    assert c.append(**kw) == _lib.SC_EINVAL
    assert _lib.last_error().startswith("sc_qwen2_paged_append: ")


def test_append_refuses_misplaced_tensors():
    c = Call()
    for name in ("q", "k", "v", "cos", "sin"):
        assert c.append(**{name: c.p + 2}) == _lib.SC_EINVAL
    for name in ("kp", "vp", "out"):
        assert c.append(**{name: c.p + 1}) == _lib.SC_EINVAL
    assert c.append(q=c.p, out=c.p) == _lib.SC_EINVAL  # in place, of another type
    assert c.append(tokens=0) == _lib.SC_OK


@pytest.mark.parametrize("kw", CACHE + [
    dict(q=None), dict(out=None), dict(out_dtype=_lib.SC_BF16), dict(out_dtype=_lib.SC_F32), dict(max_q=0), dict(max_kv=0),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(qs=255), dict(qs=257),
    dict(stride=2 * 16 * 64 + 4), dict(scratch=None)], ids=str)
def test_attention_refuses(kw):
    c = Call()
    assert c.attention(**kw) == _lib.SC_EINVAL
    assert _lib.last_error().startswith("sc_qwen2_paged_attention: ")


def test_attention_refuses_misplaced_tensors_and_small_scratch():
    c = Call()
    for name in ("q", "kp", "vp", "out", "scratch"):
        assert c.attention(**{name: c.p + 8}) == _lib.SC_EINVAL
    size = _lib.LIB.sc_qwen2_paged_attention_scratch(1, 4, 2, 64, 1, 1 << 20, _lib.SC_F16)
    assert size > 0 and c.attention(nbytes=size - 1) == _lib.SC_ENOMEM
    assert c.attention(tokens=0) == _lib.SC_OK
    assert _lib.LIB.sc_qwen2_paged_attention_scratch(1, 3, 2, 64, 1, 1 << 20, _lib.SC_F16) == 0  # refused
    assert _lib.LIB.sc_qwen2_paged_attention_scratch(1, 4, 2, 64, 1, 100, _lib.SC_F16) == 0  # none wanted


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(rows=-1), dict(rows=(1 << 20) + 1), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(begin=-1),
    dict(begin=(1 << 30) - 99), dict(x=None), dict(out=None), dict(stride=99), dict(out_stride=99),
    dict(hist=1, width=5), dict(hist=1, hlen=1, width=-1), dict(hist=1, hlen=1, width=1 << 19), dict(bptr=1, nbias=3),
    dict(bptr=1, nbias=3, bids=1), dict(bptr=1, nbias=-1), dict(mask=1, words=3, masks=2), dict(mask=1, words=4, masks=1),
    dict(mask=1, words=4, masks=-1, mrow=1), dict(mask=1, words=4, masks=2, begin=32), dict(best=1), dict(value=1)], ids=str)
def test_logits_refuse(kw):
    c = Call()
    pointers = {"hist", "hlen", "bptr", "bids", "mask", "mrow", "best", "value"}
    assert c.logits(**{k: c.p if k in pointers else v for k, v in kw.items()}) == _lib.SC_EINVAL
    assert _lib.last_error().startswith("sc_qwen2_process_logits: ")


def test_logits_refuse_misplaced_tensors_and_small_scratch():
    c = Call()
    assert c.logits(x=c.p + 2) == _lib.SC_EINVAL and c.logits(out=c.p + 1) == _lib.SC_EINVAL
    need = _lib.LIB.sc_qwen2_process_logits_scratch(2, 100)
    assert need >= 16
    assert c.logits(best=c.p, scratch=c.p, nbytes=need - 1) == _lib.SC_ENOMEM
    assert c.logits(best=c.p, scratch=c.p + 4, nbytes=need) == _lib.SC_EINVAL
    assert c.logits(rows=0) == _lib.SC_OK
    assert _lib.LIB.sc_qwen2_process_logits_scratch(0, 5) == 0 and _lib.LIB.sc_qwen2_process_logits_scratch(2, 0) == 0


def test_cache_bookkeeping():
    c = sc.PagedKVCache(2, 10, 16, 2, 64, max_seqs=3, max_positions=100, device="cpu", dtype=torch.bfloat16)
    assert len(c.k) == len(c.v) == 2 and c.k[0].shape == (10, 2, 16, 64) and c.k[0].dtype == torch.bfloat16
    assert c.block_table.shape == (3, 7) and c.free_pages == 10
    c.reserve(0, 33)
    c.reserve(1, 16)
    c.reserve(0, 40)
    assert c.pages(0) == c.block_table[0, :3].tolist() and c.pages(1) == c.block_table[1, :1].tolist()
    assert not set(c.pages(0)) & set(c.pages(1)) and c.free_pages == 6
    c.reserve(0, 49)  # a fourth page behind the three it has
    assert c.pages(0) == c.block_table[0, :4].tolist() and c.free_pages == 5
    before = c.pages(2), c.free_pages, c.block_table.clone()
    with pytest.raises(RuntimeError, match="6 pages wanted, 5 of 10 free"):
        c.reserve(2, 96)
    assert (c.pages(2), c.free_pages) == before[:2] and torch.equal(c.block_table, before[2])
    with pytest.raises(ValueError):
        c.reserve(2, 101)
    with pytest.raises(ValueError):
        c.reserve(2, -1)
    c.release(0)
    c.release(0)
    assert c.free_pages == 9 and c.pages(0) == []
    c.reserve(2, 96)
    assert len(set(c.pages(2)) | set(c.pages(1))) == 7
    for bad in (dict(page_size=24), dict(page_size=4), dict(head_dim=32), dict(num_pages=0), dict(layers=0)):
        a = dict(layers=1, num_pages=4, page_size=16, kv_heads=1, head_dim=64) | bad
        with pytest.raises(ValueError):
            sc.PagedKVCache(**a, max_seqs=1, max_positions=8, device="cpu")
    with pytest.raises(ValueError):
        sc.PagedKVCache(1, 4, 16, 1, 64, max_seqs=1, max_positions=8, device="cpu", dtype=torch.float64)
    c.check_device()
    c.status[0] = 2
    with pytest.raises(sc.CTarqError):
        c.check_device()
    c.check_device()


def test_logit_rules_refuse():
    with pytest.raises(ValueError):
        sc.LogitRules(2, "cpu", repetition=0.0)
    with pytest.raises(ValueError):
        sc.LogitRules(2, "cpu", presence=[1.0, 2.0, 3.0])
    with pytest.raises(ValueError):
        sc.LogitRules(2, "cpu", bias=[{}])
    with pytest.raises(ValueError):
        sc.LogitRules(1, "cpu", bias=[{i: 1.0 for i in range(4096)}])
    r = sc.LogitRules(3, "cpu", repetition=1.2, bias=[{4: 1.0, 2: 3.0}, {}, {9: -1.0}])
    assert r.bias_ptr.tolist() == [0, 2, 2, 3] and r.bias_ids.tolist() == [4, 2, 9]
    ptr, ids, vals = r._bias_of(torch.tensor([2, 0]))
    assert ptr.tolist() == [0, 1, 3] and ids.tolist() == [9, 4, 2] and vals.tolist() == [-1.0, 1.0, 3.0]


def test_cache_refuses_slots_it_does_not_have():
    c = sc.PagedKVCache(1, 4, 16, 1, 64, max_seqs=2, max_positions=32, device="cpu")
    for slot in (-1, 2):
        for call in (lambda: c.reserve(slot, 5), lambda: c.release(slot), lambda: c.pages(slot)):
            with pytest.raises(ValueError, match="slot"):
                call()
    assert c.free_pages == 4
