"""The attention operators' C entries without a GPU: what they refuse before
they look for a device, and that they fail loudly where there is none."""
import ctypes

import numpy as np
import pytest

import tinygiant_b200 as tg

BUF = np.zeros(1 << 14, np.float32)
P = BUF.ctypes.data


def strides(*changed):
    s = [64] * 16
    for i, x in changed:
        s[i] = x
    return (ctypes.c_int64 * 16)(*s)


def prompt(lib, dtype=0, n=1, tq=4, tk=4, max_k=4, H=4, KH=2, hd=64, st=None, window=0, scale=0.125):
    return lib.tg_attention_prompt(dtype, P, P, P, P, P, P, None, n, tq, tk, max_k, H, KH, hd, st or strides(), window,
                                   scale, None, 0, None)


def shared(lib, dtype=0, B=2, pre=4, cap=8, max_len=8, H=4, KH=2, hd=64, st=None, window=0, scale=0.125, w=None):
    return lib.tg_attention_shared(dtype, P, P, P, P, P, P, P, None, w, B, pre, cap, max_len, H, KH, hd,
                                   st or strides(), window, scale, None, 0, None)


def evict(lib, B=2, cap=8, KH=2, hd=64, st=None, keep=4, recent=1):
    return lib.tg_cache_evict(P, P, P, P, P, P, P, P, P, B, cap, KH, hd, st or strides(), keep, recent, None)


@pytest.mark.parametrize("call,bad,text", [
    (prompt, dict(dtype=2), "dtype"), (prompt, dict(tq=-1), "negative"), (prompt, dict(window=-1), "negative"),
    (prompt, dict(H=5), "multiple of n_kv_heads"), (prompt, dict(KH=0), "multiple of n_kv_heads"),
    (prompt, dict(H=129, KH=1), "128"), (prompt, dict(hd=60), "head_dim"), (prompt, dict(hd=136), "head_dim"),
    (prompt, dict(scale=float("nan")), "scale"), (prompt, dict(scale=0.0), "scale"), (prompt, dict(n=0), "sequence"),
    (prompt, dict(st=strides((3, 12))), "strides"), (prompt, dict(st=strides((0, 0))), "strides"),
    (prompt, dict(st=strides((7, -64))), "strides"),
    (shared, dict(dtype=-1), "dtype"), (shared, dict(max_len=9), "max_len"), (shared, dict(pre=-1), "negative"),
    (shared, dict(H=3), "multiple of n_kv_heads"), (shared, dict(hd=0), "head_dim"),
    (shared, dict(scale=float("inf")), "scale"), (shared, dict(st=strides((11, 4))), "strides"),
    (shared, dict(w=P, st=strides((14, 0))), "weights"),
    (evict, dict(keep=0), "keep"), (evict, dict(keep=9), "keep"), (evict, dict(recent=5), "recent"),
    (evict, dict(recent=-1), "recent"), (evict, dict(cap=0), "cap"), (evict, dict(hd=12), "head_dim"),
    (evict, dict(B=40000), "65535"), (evict, dict(st=strides((1, 20))), "strides"),
])
def test_bad_arguments_are_refused(lib, call, bad, text):
    assert call(lib, **bad) == 3
    code, msg = tg.last_error(lib)
    assert code == 3 and text in msg, msg


def test_no_device_is_an_error(lib):
    if lib.tg_cuda_device_count() > 0:
        pytest.skip("a GPU is visible")
    for call in (prompt, shared, evict):
        rc = call(lib)
        assert rc != 0 and rc == tg.last_error(lib)[0]


def test_empty_calls_need_no_device(lib):
    assert prompt(lib, tq=0) == 0 and shared(lib, B=0) == 0 and evict(lib, B=0) == 0


def test_workspace_sizes_are_monotonic(lib):
    one = lib.tg_attention_prompt_workspace(1, 8, 4096, 32, 4, 128)
    assert lib.tg_attention_prompt_workspace(4, 4096, 4096, 32, 4, 128) >= one >= 0
    few = lib.tg_attention_shared_workspace(2, 100, 64, 32, 4, 128, 0)
    assert lib.tg_attention_shared_workspace(64, 4096, 640, 32, 4, 128, 0) >= few >= 0
    assert lib.tg_attention_shared_workspace(2, 100, 64, 32, 4, 128, 1) >= few
