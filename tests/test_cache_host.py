"""What the key/value cache and log-probability entry points refuse before any device work."""

import ctypes

import pytest

from quantibbler_b200 import _lib
from quantibbler_b200._lib import QK_BF16, QK_ERR_VALUE, QK_F32, QK_F64, QK_I8, KernelError
from quantibbler_b200.cache import KvCache, KvCacheStruct

P = 4096   # a pointer that is never followed


def cache(dtype=QK_I8, k=P, v=P, ks=P, vs=P, n_seq=2, n_kv=2, rows=8, d=16):
    return KvCacheStruct(dtype, k, v, ks, vs, n_seq, n_kv, rows, d)


def refused(status, text):
    assert status == QK_ERR_VALUE
    assert text in _lib.last_error()


@pytest.mark.parametrize("change,text", [
    (dict(dtype=QK_F64), "dtype must be float32, bfloat16 or int8"),
    (dict(dtype=7), "dtype must be float32, bfloat16 or int8"),
    (dict(n_seq=0), "cache is empty"), (dict(n_kv=0), "cache is empty"), (dict(rows=0), "cache is empty"),
    (dict(d=0), "cache is empty"), (dict(d=17), "head_dim must be even and at most 256"),
    (dict(d=258), "head_dim must be even and at most 256"), (dict(rows=1 << 31), "at most 2^31 - 1 rows"),
    (dict(n_kv=65536), "65535 kv heads"), (dict(k=None), "k or v is null"), (dict(v=None), "k or v is null"),
    (dict(ks=None), "needs k_scale and v_scale"), (dict(vs=None), "needs k_scale and v_scale")])
def test_descriptions(change, text):
    lib, c = _lib.lib(), cache(**change)
    refused(lib.qk_cache_check(None, ctypes.byref(c)), text)
    refused(append(c), text)
    refused(read(c), text)
    refused(attend(c), text)
    refused(portion(c), text)


def test_null_description():
    refused(_lib.lib().qk_cache_check(None, None), "cache is null")


def append(c, q=P, q_stride=64, q_out=P, q_out_stride=64, heads=4, k=P, k_stride=32, v=P, v_stride=32, cos=P,
           n_positions=8, pos=P, seq=P, first=0, n=3):
    return _lib.lib().qk_cache_append(None, ctypes.byref(c), q, q_stride, q_out, q_out_stride, heads, k, k_stride, v,
                                      v_stride, cos, n_positions, pos, seq, first, n)


@pytest.mark.parametrize("change,text", [
    (dict(heads=3), "n_kv_heads must divide n_heads"), (dict(heads=0), "n_kv_heads must divide n_heads"),
    (dict(q_stride=63), "rows of 64 values cannot be 63 apart"), (dict(q_out=None), "q_out is null"),
    (dict(q_out_stride=1), "q_out: rows"), (dict(k=None), "k is null"), (dict(v=None), "v is null"),
    (dict(k_stride=31), "k: rows of 32"), (dict(v_stride=0), "v: rows of 32"), (dict(cos=None), "cos_sin"),
    (dict(pos=None), "positions"), (dict(seq=None), "seq_index"), (dict(n=(1 << 24) + 1), "more than one call takes"),
    (dict(first=1 << 31), "positions are 32-bit"), (dict(n_positions=1 << 31), "positions are 32-bit")])
def test_append(change, text):
    refused(append(cache(), **change), text)


def read(c, pos=P, seq=P, first=0, n=3, dtype=QK_F32, k=P, v=P):
    return _lib.lib().qk_cache_read(None, ctypes.byref(c), pos, seq, first, n, dtype, k, v)


@pytest.mark.parametrize("change,text", [
    (dict(pos=None), "is null"), (dict(seq=None), "is null"), (dict(k=None), "is null"), (dict(v=None), "is null"),
    (dict(dtype=QK_I8), "read as float32 or bfloat16"), (dict(dtype=QK_F64), "read as float32 or bfloat16"),
    (dict(first=1 << 31), "positions are 32-bit")])
def test_read(change, text):
    refused(read(cache(), **change), text)


def attend(c, prefix=None, prefix_seq=0, prefix_len=0, q=P, q_stride=64, kv_len=P, batch=2, heads=4, scratch=P, out=P,
           out_stride=64):
    p = None if prefix is None else ctypes.byref(prefix)
    return _lib.lib().qk_cache_attend(None, ctypes.byref(c), p, prefix_seq, prefix_len, q, q_stride, kv_len, batch, heads,
                                      scratch, out, out_stride)


def portion(c, seq=0, first=0, prefix=None, prefix_seq=0, prefix_len=0, q=P, q_stride=64, n=3, heads=4, scratch=P, out=P,
            out_stride=64):
    p = None if prefix is None else ctypes.byref(prefix)
    return _lib.lib().qk_cache_portion(None, ctypes.byref(c), seq, first, p, prefix_seq, prefix_len, q, q_stride, n, heads,
                                       scratch, out, out_stride)


PREFIXES = [
    (dict(prefix_len=1), "prefix is null"),
    (dict(prefix_len=1, prefix=cache(dtype=QK_BF16)), "agree in dtype"),
    (dict(prefix_len=1, prefix=cache(n_kv=4)), "agree in dtype"), (dict(prefix_len=1, prefix=cache(d=32)), "agree in dtype"),
    (dict(prefix_len=9, prefix=cache()), "do not lie in 2 slots of 8 rows"),
    (dict(prefix_len=1, prefix_seq=2, prefix=cache()), "do not lie in 2 slots of 8 rows"),
    (dict(prefix_len=1, prefix=cache(ks=None)), "needs k_scale")]


@pytest.mark.parametrize("change,text", PREFIXES + [
    (dict(batch=3), "the cache has 2 slots"), (dict(heads=5), "n_kv_heads must divide n_heads"), (dict(q=None), "q is null"),
    (dict(out=None), "out is null"), (dict(q_stride=32), "q: rows of 64"), (dict(out_stride=63), "out: rows of 64"),
    (dict(kv_len=None), "kv_len is null"), (dict(wide=True, scratch=None), "scratch is null"),
    (dict(wide=True, scratch=P + 8), "no 16-byte boundary"), (dict(heads=1 << 17), "more than one call takes")])
def test_attend(change, text):
    change = dict(change)
    if change.pop("wide", False):   # a shape whose keys are split over blocks
        refused(attend(cache(rows=200_000, d=128), q_stride=512, out_stride=512, **change), text)
    else:
        refused(attend(cache(), **change), text)


@pytest.mark.parametrize("change,text", PREFIXES + [
    (dict(seq=2), "slot 2 outside"), (dict(first=6), "do not fit the cache of 8 rows"), (dict(n=9), "do not fit"),
    (dict(first=9, n=0), "do not fit"), (dict(first=(1 << 64) - 2), "do not fit"), (dict(q=None), "q is null"),
    (dict(out_stride=1), "out: rows of 64"), (dict(heads=3), "n_kv_heads must divide")])
def test_portion(change, text):
    refused(portion(cache(), **change), text)


def log_probs(logits=P, n=2, vocab=100, stride=100, targets=P, top=5, scratch=P, lse=P, logprob=P):
    return _lib.lib().qk_log_probs(None, logits, n, vocab, stride, targets, top, scratch, lse, logprob, P, P, P)


@pytest.mark.parametrize("change,text", [
    (dict(vocab=0), "vocab must lie in"), (dict(vocab=1 << 31, stride=1 << 31), "vocab must lie in"),
    (dict(stride=99), "rows of 100 logits"), (dict(top=33), "n_top must be at most 32"),
    (dict(vocab=4, top=5), "n_top must be at most"), (dict(logits=None), "logits is null"),
    (dict(targets=None), "logprob needs targets"), (dict(n=(1 << 24) + 1), "more than one call takes")])
def test_log_probs(change, text):
    refused(log_probs(**change), text)


def test_tensors_of_another_device():
    import torch
    from quantibbler_b200.scoring import log_probs as scored

    class Ctx:   # (no device is touched: the checks come first)
        device_index, handle = 0, None

    z = torch.zeros(1, 1, 4, 16)
    with pytest.raises(KernelError, match="lives on a CUDA device"):
        KvCache(Ctx, z, z)
    with pytest.raises(KernelError, match="holds float32, bfloat16 or int8"):
        KvCache(Ctx, z.double(), z.double())
    with pytest.raises(KernelError, match="k must be"):
        KvCache(Ctx, z[0], z[0])
    with pytest.raises(KernelError, match="cache dtype must be one of"):
        KvCache.empty(Ctx, 1, 1, 4, 16, dtype="float16")
    with pytest.raises(KernelError, match="logits are on cpu"):
        scored(Ctx, torch.zeros(2, 8))
    with pytest.raises(KernelError, match="logits must be"):
        scored(Ctx, torch.zeros(8))
