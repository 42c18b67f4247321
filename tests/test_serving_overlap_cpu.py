"""Outputs that lie over inputs in another way than in place are refused, without a GPU."""
import ctypes

import pytest

pytest.importorskip("torch")

from saccade_core import _lib
from test_paged_cpu import Call, _buf

ROW, KV = 4 * 64, 2 * 64  # elements of a token's queries and keys


def refused(status, what):
    assert status == _lib.SC_EINVAL and what in _lib.last_error(), _lib.last_error()


@pytest.fixture
def call():
    c = Call()
    c.far = _buf()  # kept alive: another buffer
    return c


# In these calls everything else passes: what is allowed then stops at the scratch that is too small.

def test_attention_over_its_queries(call):
    at = lambda **kw: call.attention(nbytes=0, **kw)  # noqa: E731
    assert at() == _lib.SC_ENOMEM                                     # in place
    assert at(out=call.p + 4 * ROW * 2) == _lib.SC_ENOMEM             # right behind them
    assert at(tokens=1, qs=ROW * 3) == _lib.SC_ENOMEM                 # one row has no stride
    assert at(out=call.far[1], qs=ROW * 2) == _lib.SC_ENOMEM
    refused(at(qs=ROW * 2), "out over q")                             # rows move
    refused(at(out=call.p + 16), "out over q")
    refused(at(out=call.p + 4 * ROW * 2 - 16), "out over q")
    refused(at(q=call.p + 4 * ROW * 2 - 16), "out over q")
    refused(at(dtype=_lib.SC_F32, out_dtype=_lib.SC_F16), "out over q")
    refused(at(dtype=_lib.SC_F32, out_dtype=_lib.SC_F16, tokens=1), "out over q")


def test_append_over_its_inputs(call):
    size, far = 4 * ROW * 2, call.far[1]
    f16 = dict(in_dtype=_lib.SC_F16, k=far, v=far)
    bad = dict(max_pos=0)  # refused before: what the others are told comes later
    refused(call.append(**f16, **bad), "empty rotation tables")
    refused(call.append(k=far, v=far), "in place")                    # f32 queries
    refused(call.append(**f16, qs=ROW * 2), "in place")
    refused(call.append(**f16, out=call.p + 16), "in place")
    refused(call.append(**f16, out=call.p + size - 16), "in place")
    refused(call.append(**f16, q=call.p + size - 16), "in place")
    refused(call.append(**(f16 | dict(k=call.p + size - 16))), "over k or v")
    refused(call.append(**(f16 | dict(v=call.p + size - 2))), "over k or v")
    # a call with nothing of that wrong gets to the alignment of its tables
    refused(call.append(**f16, cos=far + 2), "aligned")
    refused(call.append(**(f16 | dict(k=call.p + size, v=call.p + size)), cos=far + 2), "aligned")
    refused(call.append(**f16, q=call.p + size, cos=far + 2), "aligned")


def test_logits_over_their_inputs(call):
    p = call.p
    lg = lambda **kw: call.logits(best=p, scratch=p, nbytes=0, **kw)  # noqa: E731
    ok = _lib.SC_ENOMEM
    assert lg() == ok                                                 # in place
    assert lg(out=p + 800) == ok                                      # behind
    assert lg(stride=200, out_stride=200, out=p + 400) == ok          # columns beside each other
    assert lg(stride=200, out_stride=200, out=p + 400 + 800) == ok
    assert lg(stride=200, out_stride=200, x=p + 400) == ok
    assert lg(stride=300, out_stride=300, out=p + 500) == ok
    assert lg(rows=1, stride=5, out_stride=7) == ok                   # one row has no stride
    refused(lg(stride=200), "another stride")
    refused(lg(out_stride=101), "another stride")
    refused(lg(out=p + 4), "not in place")
    refused(lg(out=p + 400), "not in place")                          # the second row
    refused(lg(x=p + 796), "not in place")
    refused(lg(rows=1, out=p + 396), "not in place")
    refused(lg(rows=1, x=p + 4), "not in place")
    refused(lg(stride=200, out_stride=200, out=p + 396), "not in place")
    refused(lg(stride=200, out_stride=200, x=p + 404), "not in place")
    refused(lg(stride=300, out_stride=300, out=p + 804), "not in place")
