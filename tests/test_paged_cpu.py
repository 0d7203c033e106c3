"""The paged cache without a GPU: where tokens lie (csrc/tg_paged.h, compiled
for the host with the sanitizers of bounds and undefined behaviour, tables and
offsets of garbage among its inputs), frequencies against their definition,
and what the C entries refuse before they look for a device."""
import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import tinygiant_b200 as tg

torch = pytest.importorskip("torch")
CSRC = Path(__file__).resolve().parents[1] / "tinygiant_b200" / "csrc"
MAIN = r"""
#include "tg_paged.h"
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>
using namespace tg;
#define NEED(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
  // pages: every place or none, for numbers of any kind
  const int odd[] = {0, 1, 4, 5, -1, -7, 1 << 30, 0x7fffffff, (int)0x80000000};
  for (int shift : {4, 5, 8})
    for (int n_pages : {0, 1, 5})
      for (int cols : {0, 1, 9}) {
        std::vector<int> table(cols);
        for (int i = 0; i < cols; i++) table[i] = odd[i];
        for (long long p : {-0x80000000ll, -17ll, -1ll, 0ll, 15ll, 16ll, 143ll, 144ll, 255ll, 256ll, 0x7fffffffll}) {
          const int got = paged_page(table.data(), cols, (int)p, shift, n_pages);
          const bool in = p >= 0 && (p >> shift) < cols && table[p >> shift] >= 0 && table[p >> shift] < n_pages;
          NEED(got == (in ? table[p >> shift] : -1));
        }
      }
  // tokens: ascending offsets
  {
    const int cu[] = {2, 2, 5, 5, 9, 12};
    const int seq[] = {-1, -1, 1, 1, 1, 3, 3, 3, 3, 4, 4, -1, -1};
    for (int t = 0; t < 13; t++) {
      const PagedToken k = paged_token(cu, 5, 1, 11, t);
      const int want = t < 11 ? seq[t] : -1;
      NEED(k.seq == want);
      if (want >= 0) NEED(k.first <= t && t < k.end && k.end <= 11);
    }
    for (int t = 0; t < 12; t++) {
      const PagedToken k = paged_token(nullptr, 4, 3, 12, t);
      NEED(k.seq == t / 3 && k.first == t / 3 * 3 && k.end == k.first + 3);
    }
  }
  // and of garbage: within bounds, a run within its sequence and block
  std::srand(1);
  for (int round = 0; round < 20000; round++) {
    const int n = 1 + std::rand() % 6, total = std::rand() % 40;
    std::vector<int> cu(n + 1);
    for (int& x : cu) x = std::rand() % 4 ? std::rand() % 44 - 2 : odd[std::rand() % 9];
    for (int t = 0; t < total; t++) {
      const PagedToken k = paged_token(cu.data(), n, 1, total, t);
      NEED(k.seq >= -1 && k.seq < n);
      if (k.seq < 0) continue;
      NEED(k.first >= 0 && k.first <= t && t < k.end && k.end <= total);
      for (int len : {0, 1, 7, 33, odd[std::rand() % 9], std::rand()}) {
        const int p = paged_position(len, k.end, t), r = paged_run(k, t, p);
        NEED((long long)p == std::max((long long)len - (k.end - t), -0x7fffffffll));
        NEED(r >= 0 && t + r <= k.end && (r == 0 || (p >= 0 && p % 16 + r <= 16)));
      }
    }
  }
  // runs cover each token with a place once
  for (int len : {1, 5, 16, 17, 40, 300})
    for (int n : {1, 2, 16, 40, 300}) {
      std::vector<int> seen(n);
      const PagedToken k{0, 0, n};
      for (int t = 0; t < n; t++)
        for (int i = 0, r = paged_run(k, t, paged_position(len, n, t)); i < r; i++) seen[t + i]++;
      for (int t = 0; t < n; t++) NEED(seen[t] == (len - n + t >= 0));
    }
  // scales: the least power of two under which the value is at most 448
  for (int i = 0; i < 2000000; i++) {
    uint32_t bits = i < 1000 ? (uint32_t)i : ((uint32_t)std::rand() << 8 ^ (uint32_t)std::rand()) & 0x7fffffffu;
    if (i >= 1000 && i < 5000) bits = ((uint32_t)(i % 250 + 2) << 23 | 0x600000u) + (i / 250) % 3 - 1;
    if (bits >= 0x7f800000u) continue;
    float x;
    std::memcpy(&x, &bits, 4);
    const int e = paged_scale_exp(bits);
    NEED(e >= -117 && e <= 120);
    NEED((double)x <= 448 * std::ldexp(1.0, e));
    if (e > -117) NEED((double)x > 448 * std::ldexp(1.0, e - 1));
  }
  // tiles: all keys that the queries read, from a whole block on
  for (int len : {0, 1, 15, 16, 17, 128, 1000, 0x3ffffffe})
    for (int q : {1, 2, 8, 5000})
      for (int w : {0, 1, 15, 128, 999, 0x7fffffff})
        for (int keys : {16, 32}) {
          const int lo = paged_first(len, q, w), n = paged_tiles(len, q, w, keys);
          const long long first = w ? std::max(0ll, (long long)len - q + 1 - w) : 0;
          NEED(lo == first);
          NEED(len == 0 ? n == 0 : lo < len ? (long long)(lo & ~15) + (long long)n * keys >= len && (long long)(lo & ~15) + (n - 1ll) * keys < len : true);
        }
  std::puts("ok");
}
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="no g++")
def test_places_of_tokens(tmp_path):
    src, exe = tmp_path / "main.cpp", tmp_path / "main"
    src.write_text("#include <algorithm>\n" + MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined,address", "-fno-sanitize-recover=all", "-D_GLIBCXX_ASSERTIONS",
                    "-I", str(CSRC), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_frequencies():
    from tinygiant_b200.paged import rotary_frequencies as F
    f, s = F(128, 1e6)
    assert f.dtype == torch.float64 and s == 1.0
    assert np.allclose(f.numpy(), 1e6 ** (-np.arange(64) / 64), rtol=1e-15, atol=0)
    assert np.allclose(F(64, 1e4, scaling="linear", factor=8)[0].numpy(), 1e4 ** (-np.arange(32) / 32) / 8, rtol=1e-15, atol=0)
    ntk = F(64, 1e4, scaling="ntk", factor=4)[0].numpy()
    assert ntk[0] == 1 and math.isclose(ntk[-1], 1e4 ** (-31 / 32) / 4, rel_tol=1e-12)   # the slowest turns a quarter as fast
    plain = 150000.0 ** (-np.arange(32) / 32)
    f, s = F(64, 150000.0, scaling="yarn", factor=32, original_len=4096)
    assert math.isclose(s, 0.1 * math.log(32) + 1)
    turns = 4096 * plain / (2 * math.pi)
    ratio = plain / f.numpy()
    assert np.all(ratio[turns > 64] == 1) and np.allclose(ratio[turns < 0.5], 32, rtol=1e-12) and np.all(np.diff(ratio) >= 0)
    # the ramp between the pairs that turn 32 times and once, its ends whole pairs or not
    ends = 64 * np.log(4096 / (np.array([32, 1]) * 2 * math.pi)) / (2 * math.log(150000.0))
    for truncate, (low, high) in ((True, (math.floor(ends[0]), math.ceil(ends[1]))), (False, ends)):
        w = np.clip((np.arange(32) - low) / (high - low), 0, 1)
        got = F(64, 150000.0, scaling="yarn", factor=32, original_len=4096, truncate=truncate)[0].numpy()
        assert np.allclose(got, plain / 32 * w + plain * (1 - w), rtol=1e-13, atol=0)
    assert F(64, 1e4, scaling="yarn", factor=1, original_len=4096)[1] == 1.0
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, theta=1.0), dict(dim=8, factor=0.5), dict(dim=8, scaling="other"),
                dict(dim=8, scaling="yarn", factor=2), dict(dim=2, scaling="ntk", factor=2), dict(dim=8, theta=math.nan)):
        with pytest.raises(ValueError):
            F(**bad)


BUF = np.zeros(1 << 14, np.float32)
P = BUF.ctypes.data


def strides(*changed, n=21):
    s = [64] * n
    for i, x in changed:
        s[i] = x
    return (ctypes.c_int64 * n)(*s)


def rot(lib, dtype=0, T=4, H=4, KH=2, hd=64, nf=32, amp=1.0, eps=1e-6, st=None):
    return lib.tg_rotary(dtype, P, P, P, P, P, P, None, None, T, H, KH, hd, nf, 0, amp, eps, st or strides(), None)


def append(lib, dtype=0, bits=16, T=4, B=2, N=3, page=16, cols=2, H=4, KH=2, hd=64, nf=32, amp=1.0, eps=1e-6, st=None, cu=P):
    return lib.tg_paged_append(dtype, bits, P, P, P, P, P, P, P, P, P, P, cu, None, P, None, None, T, B, N, page, cols, H, KH, hd, nf, 0,
                               amp, eps, st or strides(), None)


def attn(lib, dtype=0, bits=16, B=2, n=1, N=3, page=16, cols=2, max_len=32, H=4, KH=2, hd=64, st=None, window=0, scale=0.125):
    return lib.tg_attention_paged(dtype, bits, P, P, P, P, P, P, P, P, None, B, n, N, page, cols, max_len, H, KH, hd, st or strides(),
                                  window, scale, None, 0, None)


def gather(lib, dtype=0, bits=16, total=4, B=2, N=3, page=16, cols=2, KH=2, hd=64, st=None):
    return lib.tg_paged_gather(dtype, bits, P, P, P, P, P, P, P, P, total, B, N, page, cols, KH, hd, st or strides(), None)


POOL = [(dict(bits=4), "page_bits"), (dict(page=8), "page must be"), (dict(page=48), "page must be"), (dict(page=0), "page must be"),
        (dict(N=-1), "n_pages"), (dict(cols=-1), "table_cols"), (dict(bits=8, hd=72), "multiple of 16"), (dict(hd=60), "head_dim"),
        (dict(hd=136), "head_dim"), (dict(dtype=2), "dtype")]


@pytest.mark.parametrize("call,bad,text", [(c, b, t) for c in (append, attn, gather) for b, t in POOL] + [
    (rot, dict(dtype=5), "dtype"), (rot, dict(T=-1), "negative"), (rot, dict(hd=12), "head_dim"), (rot, dict(nf=33), "frequencies"),
    (rot, dict(amp=math.inf), "amplitude"), (rot, dict(eps=-1.0), "eps"), (rot, dict(eps=math.nan), "eps"),
    (rot, dict(st=strides((1, 12))), "strides"), (rot, dict(st=strides((6, 0))), "strides"),
    (append, dict(KH=0), "n_kv_heads"), (append, dict(T=3, cu=None), "as many"), (append, dict(B=0), "without a sequence"),
    (append, dict(nf=-1), "frequencies"), (append, dict(st=strides((4, 4))), "strides"), (append, dict(st=strides((10, 4))), "pages"),
    (append, dict(bits=8, st=strides((8, 72))), "pages"), (append, dict(bits=8, page=32, st=strides((16, 0))), "scales"),
    (append, dict(st=strides((20, 0))), "tables"), (append, dict(amp=math.nan), "amplitude"),
    (attn, dict(H=5), "multiple of n_kv_heads"), (attn, dict(H=258), "128"), (attn, dict(window=-1), "negative"),
    (attn, dict(max_len=33), "max_len"), (attn, dict(scale=0.0), "scale"), (attn, dict(scale=math.nan), "scale"),
    (attn, dict(n=-1), "negative"), (attn, dict(n=1 << 23), "rows"), (attn, dict(cols=1 << 30, max_len=0x3fffffff), "positions"),
    (attn, dict(st=strides((5, 20))), "strides"), (attn, dict(st=strides((6, -64))), "pages"), (attn, dict(st=strides((18, -1))), "tables"),
    (gather, dict(total=-1), "negative"), (gather, dict(KH=0), "n_kv_heads"), (gather, dict(st=strides((2, 4))), "strides"),
    (gather, dict(bits=8, page=32, st=strides((12, -1))), "scales"),
])
def test_bad_arguments_are_refused(lib, call, bad, text):
    assert call(lib, **bad) == 3
    code, msg = tg.last_error(lib)
    assert code == 3 and text in msg, msg


def test_no_device_is_an_error(lib):
    if lib.tg_cuda_device_count() > 0:
        pytest.skip("a GPU is visible")
    for call in (rot, append, attn, gather):
        rc = call(lib)
        assert rc != 0 and rc == tg.last_error(lib)[0]


def test_empty_calls_need_no_device(lib):
    assert rot(lib, T=0) == 0 and rot(lib, H=0, KH=0) == 0 and append(lib, T=0) == 0 and append(lib, T=0, B=0) == 0
    assert attn(lib, B=0) == 0 and attn(lib, n=0) == 0 and gather(lib, total=0) == 0 and gather(lib, B=0) == 0


def test_python_refuses_what_is_on_the_host():
    from tinygiant_b200 import paged
    q, f = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(32, dtype=torch.float64)
    i, pages = torch.zeros(3, dtype=torch.int32), torch.zeros(2, 4, 16, 64, dtype=torch.bfloat16)
    for call in (lambda: paged.rotary(q, None, i, f), lambda: paged.rotary(None, None, i, f), lambda: paged.rotary(q.float(), None, i, f),
                 lambda: paged.cache_append(q, q, pages, pages, i[:, None], i), lambda: paged.cache_append(None, q, pages, pages, i, i),
                 lambda: paged.attention_paged(q, pages, pages, i[:, None], i), lambda: paged.attention_paged(None, pages, pages, i, i),
                 lambda: paged.cache_gather(pages, pages, i[:, None], i, 3), lambda: paged.cache_gather(None, None, None, None, 3)):
        with pytest.raises(ValueError):
            call()
