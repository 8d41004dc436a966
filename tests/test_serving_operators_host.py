"""Refusals of the operators on the paged cache and of the log probabilities, on the CPU: every argument is checked before a pointer is
used or anything is launched."""
import ctypes

import pytest

import garnet_b200
from garnet_b200 import _lib, cache, decode as dec

P = 4096                                   # stands for a device pointer; never followed


def chunk_options(**kw):
    base = dict(abi=1, struct_size=ctypes.sizeof(dec.AttentionOptions), q_heads=4, kv_heads=2, head_dim=128, page_size=16, max_logical_pages=8,
                max_context=128, rope_positions=128, norm_eps=1e-6)
    return dec.AttentionOptions(**dict(base, **kw))


def chunk(opt, ws=P, ws_bytes=1 << 30, batch=1, tokens=4, pages=8, **ptr):
    p = {n: P for n in ("qkv", "qn", "kn", "cos", "sin", "k", "v", "table", "positions", "starts", "out")}
    p.update(ptr)
    return garnet_b200.lib().garnet_b200_attention_chunk(ctypes.byref(opt), p["qkv"], p["qn"], p["kn"], p["cos"], p["sin"], p["k"], p["v"], p["table"],
                                                         p["positions"], p["starts"], p["out"], ws, ws_bytes, batch, tokens, pages, 0, None)


def test_chunk_options():
    n = ctypes.c_size_t(0)
    L = garnet_b200.lib()
    assert L.garnet_b200_attention_chunk_workspace(ctypes.byref(chunk_options()), 5, ctypes.byref(n)) == _lib.OK and n.value > 0
    one = n.value
    assert L.garnet_b200_attention_chunk_workspace(ctypes.byref(chunk_options()), 50, ctypes.byref(n)) == _lib.OK and n.value > one
    for code, kw in ((_lib.INVALID_VALUE, dict(abi=2)), (_lib.INVALID_VALUE, dict(struct_size=4)), (_lib.INVALID_VALUE, dict(q_heads=3)),
                     (_lib.INVALID_VALUE, dict(kv_heads=0)), (_lib.INVALID_VALUE, dict(page_size=0)), (_lib.INVALID_VALUE, dict(max_context=129)),
                     (_lib.INVALID_VALUE, dict(rope_positions=100)), (_lib.INVALID_VALUE, dict(norm_eps=0.0)), (_lib.INVALID_VALUE, dict(norm_eps=float("nan"))),
                     (_lib.NOT_SUPPORTED, dict(head_dim=64)), (_lib.NOT_SUPPORTED, dict(q_heads=258, kv_heads=2))):
        opt = chunk_options(**kw)
        assert L.garnet_b200_attention_chunk_workspace(ctypes.byref(opt), 5, ctypes.byref(n)) == code, kw
        assert chunk(opt) == code, kw
    for args in ((None, 5, ctypes.byref(n)), (ctypes.byref(chunk_options()), 0, ctypes.byref(n)), (ctypes.byref(chunk_options()), 5, None)):
        assert L.garnet_b200_attention_chunk_workspace(*args) == _lib.INVALID_VALUE


@pytest.mark.parametrize("kw", [dict(batch=0), dict(tokens=0), dict(pages=0), dict(ws=None), dict(ws=P + 16), dict(ws_bytes=4), dict(qkv=P + 8), dict(out=P + 2),
                                dict(k=P + 4), dict(v=P + 8), dict(cos=P + 4), dict(qn=P + 2)] +
                         [{n: None} for n in ("qkv", "qn", "kn", "cos", "sin", "k", "v", "table", "positions", "starts", "out")])
def test_chunk_arguments(kw):
    assert chunk(chunk_options(), **kw) == _lib.INVALID_VALUE
    assert b"attention_chunk" in garnet_b200.lib().garnet_b200_last_error()


def log_probs(logits=P, dtype=_lib.BF16, stride=100, targets=P, rows=2, vocab=100, k=3, temperature=1.0, lp=P, ranks=P, entropy=P, top=P, ids=P):
    return garnet_b200.lib().garnet_b200_log_probs(logits, dtype, stride, targets, rows, vocab, k, temperature, lp, ranks, entropy, top, ids, 0, None)


@pytest.mark.parametrize("code,kw", [(1, dict(logits=None)), (1, dict(dtype=3)), (1, dict(dtype=-1)), (1, dict(stride=99)), (1, dict(rows=0)), (1, dict(vocab=0)), (1, dict(k=-1)),
                                     (1, dict(k=101)), (2, dict(k=33)), (1, dict(temperature=0.0)), (1, dict(temperature=-1.0)), (1, dict(temperature=float("nan"))),
                                     (1, dict(temperature=float("inf"))), (1, dict(temperature=1e-45)), (1, dict(targets=None)), (1, dict(lp=None)), (1, dict(ranks=None)),
                                     (1, dict(top=None)), (1, dict(ids=None)), (1, dict(logits=P + 1)), (1, dict(logits=P + 2, dtype=_lib.FP32))])
def test_log_probs_arguments(code, kw):
    assert log_probs(**kw) == code
    assert b"log_probs" in garnet_b200.lib().garnet_b200_last_error()


def cache_options(**kw):
    base = dict(abi=1, struct_size=ctypes.sizeof(cache.CacheOptions), layers=2, physical_pages=10, page_size=16, token_bytes=512, sequences=4, max_logical_pages=4)
    return cache.CacheOptions(**dict(base, **kw))


def test_cache_arguments():
    L = garnet_b200.lib()
    n = ctypes.c_size_t(0)
    o = cache_options()
    assert L.garnet_b200_cache_workspace(ctypes.byref(o), 4, ctypes.byref(n)) == _lib.OK
    ws = n.value
    two, hole, odd = (ctypes.c_void_p * 2)(P, P), (ctypes.c_void_p * 2)(P, None), (ctypes.c_void_p * 2)(P, P + 8)
    r = ctypes.byref
    calls = {
        "extend": lambda o=o, t=P, l=P, c=P, a=P, b=P, s=P, n=4, w=P, z=ws, k=two, v=two: L.garnet_b200_cache_extend(r(o), t, l, c, a, b, s, n, w, z, None),
        "fork": lambda o=o, t=P, l=P, c=P, a=P, b=P, s=P, n=4, w=P, z=ws, k=two, v=two: L.garnet_b200_cache_fork(r(o), k, v, t, l, c, a, b, s, n, w, z, None),
        "free": lambda o=o, t=P, l=P, c=P, a=P, b=P, s=P, n=4, w=P, z=ws, k=two, v=two: L.garnet_b200_cache_free(r(o), t, l, c, a, n, None),
        "compact": lambda o=o, t=P, l=P, c=P, a=P, b=P, s=P, n=4, w=P, z=ws, k=two, v=two: L.garnet_b200_cache_compact(r(o), k, v, t, c, s, w, z, None),
        "copy_pages": lambda o=o, t=P, l=P, c=P, a=P, b=P, s=P, n=4, w=P, z=ws, k=two, v=two: L.garnet_b200_cache_copy_pages(r(o), k, v, a, b, n, None),
    }
    takes = {"extend": "tlcabsnwz", "fork": "tlcabsnwzkv", "free": "tlcan", "compact": "tcswzkv", "copy_pages": "abnkv"}
    wrong = dict(t=[None], l=[None], c=[None], a=[None], b=[None], s=[None], n=[0, -1], w=[None, P + 16], z=[0], k=[None, hole, odd], v=[None, hole, odd])
    for name, call in calls.items():
        for arg in takes[name]:
            for value in wrong[arg]:
                assert call(**{arg: value}) == _lib.INVALID_VALUE, (name, arg, value)
                assert b"cache_" + name.encode() in L.garnet_b200_last_error()
        for kw in (dict(abi=0), dict(struct_size=8), dict(layers=0), dict(physical_pages=0), dict(page_size=0), dict(token_bytes=0), dict(token_bytes=24), dict(sequences=0),
                   dict(max_logical_pages=0)):
            assert call(o=cache_options(**kw)) == _lib.INVALID_VALUE, (name, kw)
        for kw in (dict(layers=129), dict(page_size=1 << 20, token_bytes=1 << 12)):
            assert call(o=cache_options(**kw)) == _lib.NOT_SUPPORTED, (name, kw)
    assert L.garnet_b200_cache_workspace(ctypes.byref(o), -1, ctypes.byref(n)) == _lib.INVALID_VALUE
    assert L.garnet_b200_cache_workspace(None, 1, ctypes.byref(n)) == _lib.INVALID_VALUE
