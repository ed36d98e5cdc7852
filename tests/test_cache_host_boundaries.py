"""Addresses that lie on no boundary of their type are refused before any device work (a kernel's access would fault)."""

import ctypes

import pytest

from quantibbler_b200 import _lib
from quantibbler_b200._lib import QK_BF16, QK_F32, QK_I8
from tests.test_cache_host import P, append, attend, cache, log_probs, portion, read, refused


@pytest.mark.parametrize("change", [dict(dtype=QK_F32, k=P + 2), dict(dtype=QK_F32, v=P + 1), dict(dtype=QK_BF16, k=P + 1),
                                    dict(dtype=QK_BF16, v=P + 3), dict(ks=P + 2), dict(vs=P + 1)])
def test_rows_and_scales(change):
    c = cache(**change)
    for status in (_lib.lib().qk_cache_check(None, ctypes.byref(c)), append(c), read(c), attend(c), portion(c)):
        refused(status, "cache: rows or scales lie on no boundary")
    refused(attend(cache(dtype=c.dtype), prefix=c, prefix_len=1), "prefix: rows or scales lie on no boundary")


def test_codes_lie_anywhere():
    c = cache(dtype=QK_I8, k=P + 1, v=P + 3)
    refused(attend(c, kv_len=None), "kv_len is null")     # (the cache itself is taken)


@pytest.mark.parametrize("call,change,text", [
    (append, dict(q=P + 2), "q lies on no float boundary"), (append, dict(q_out=P + 1), "q_out lies on no float boundary"),
    (append, dict(k=P + 3), "k lies on no float boundary"), (append, dict(v=P + 2), "v lies on no float boundary"),
    (append, dict(cos=P + 2), "no boundary of its type"), (append, dict(pos=P + 1), "no boundary of its type"),
    (append, dict(seq=P + 2), "no boundary of its type"),
    (read, dict(pos=P + 2), "no boundary of its type"), (read, dict(seq=P + 1), "no boundary of its type"),
    (read, dict(k=P + 2), "no boundary of its type"), (read, dict(v=P + 1, dtype=QK_BF16), "no boundary of its type"),
    (attend, dict(q=P + 1), "q lies on no float boundary"), (attend, dict(out=P + 2), "out lies on no float boundary"),
    (attend, dict(kv_len=P + 2), "kv_len lies on no boundary"), (portion, dict(q=P + 3), "q lies on no float boundary"),
    (portion, dict(out=P + 1), "out lies on no float boundary")])
def test_arguments(call, change, text):
    refused(call(cache(), **change), text)


@pytest.mark.parametrize("change", [dict(targets=P + 2), dict(lse=P + 1), dict(logprob=P + 3)])
def test_log_probs(change):
    refused(log_probs(**change), "targets or an output lies on no boundary")
