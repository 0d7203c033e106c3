"""The paged cache where it can go wrong: values that are not finite beside cuts, codes and scales next to a border,
earlier scales of any kind, the C entries by their argument lists, and what is refused beside the ordinary.

Tolerances: none.  Codes, scales and NaN are compared for equality; expected codes are worked out on the host in
numpy's long doubles (64 bits of mantissa; angles reduced in decimals), from inputs chosen so that the exact value is 2^-44
of itself or more away from the border between two codes, which that arithmetic (2^-58 of a pair) and fp64's (2^-50)
resolve."""
import ctypes
import decimal
import math

import numpy as np
import pytest

import tinygiant_b200 as tg
from test_gpu_paged import DT, E4M3, Pool, bits, check, ends, gen, ints, paged_ref, rand

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
L = np.longdouble


@pytest.fixture(scope="module")
def P(gpu):
    from tinygiant_b200 import paged
    return paged


# ---- attention: what is not finite

def put(pool, x, b, j, value, kh=0, d=slice(None)):
    """A value at position j of sequence b."""
    pages = getattr(pool, x)
    pages[int(pool.tables[b, j // pool.page]), kh, j % pool.page, d] = torch.tensor(value, device="cuda").to(pages.dtype)


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("with_sinks", [False, True], ids=["plain", "sinks"])
def test_a_key_of_nan_wherever_units_are_cut(P, codes, with_sinks):
    """The newest key, alone in its tile or not, alone in its sequence's last piece or not: its sequence is NaN, the other as it was."""
    g, H, hd = gen(51), 4, 128
    sinks = torch.randn(H, generator=g, device="cuda") if with_sinks else None
    for m in [897, 898, *range(513, 1600, 32), 3009, 8193]:
        pool = Pool(g, torch.bfloat16, codes, 1, hd, 64, [m, m])
        q = rand(g, 2, H, hd, dtype=torch.bfloat16)
        for window in (0, 300):
            call = lambda: P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, sinks=sinks, max_len=m, window=window)  # noqa: E731
            clean = call()
            assert bool(torch.isfinite(clean).all())
            kept = pool.k.clone()
            for b in (0, 1):
                put(pool, "k", b, m - 1, math.nan)
                got = call()
                assert bool(torch.isnan(got[b]).all()) and torch.equal(got[1 - b], clean[1 - b]), (m, b, window)
                pool.k.copy_(kept)


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_a_key_of_nan_alone_before_a_cut(P, codes):
    """A window that begins with the last key of a tile, which is NaN: the first piece may see no other."""
    g, H, hd, n = gen(52), 4, 128, 2
    for m in range(1500, 1500 + 64, 5):
        pool = Pool(g, torch.float16, codes, 1, hd, 64, [m, m])
        q = rand(g, 2, n, H, hd, dtype=torch.float16)
        for first in (15, 31, 47):                                  # the first key that the last query sees
            window = m - first
            call = lambda: P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, max_len=m, window=window)  # noqa: E731
            clean, kept = call(), pool.k.clone()
            put(pool, "k", 1, first, math.nan)
            got = call()
            assert bool(torch.isnan(got[1]).all()) and torch.equal(got[0], clean[0]), (m, first)
            pool.k.copy_(kept)
            put(pool, "k", 1, first - 1, math.nan)                  # which the first query sees alone
            got = call()
            assert bool(torch.isnan(got[1, 0]).all()) and torch.equal(got[1, 1:], clean[1, 1:]) and torch.equal(got[0], clean[0])
            pool.k.copy_(kept)


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_a_query_of_nan_over_long_sequences(P, codes):
    g, H, KH, hd, lens = gen(53), 8, 2, 64, [5000, 700, 2048, 33]
    pool = Pool(g, torch.bfloat16, codes, KH, hd, 16, lens)
    q = rand(g, 4, 1, H, hd, dtype=torch.bfloat16)
    for sinks in (None, torch.randn(H, generator=g, device="cuda")):
        call = lambda: P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, sinks=sinks)  # noqa: E731
        q[:, 0, 3] = 1.0
        clean = call()
        check(clean, *paged_ref(pool, q, lens, 0, sinks), codes)
        q[:, 0, 3, 5] = math.nan
        got = call()
        assert bool(torch.isnan(got[:, 0, 3]).all())
        keep = [h for h in range(H) if h != 3]
        assert torch.equal(got[:, :, keep], clean[:, :, keep])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("m", [90, 400, 3000, 20000])
def test_values_of_nan_under_weights_that_vanish(P, m, codes, dtype):
    """A value of NaN whose weight is 2^-300 of the largest reaches its dimension, whichever warp, piece or tile has it."""
    g, hd, dt = gen(54), 64, DT[dtype]
    pool = Pool(g, dt, codes, 1, hd, 16, [m])
    pool.k.copy_(torch.zeros_like(pool.k, dtype=torch.float32).to(pool.k.dtype))
    if codes:
        pool.ks[:] = 1.0
    q = torch.zeros(1, 1, 2, hd, dtype=dt, device="cuda")
    q[..., 0] = 20.0
    top = m // 3
    put(pool, "k", 0, top, 15.0, d=0)
    call = lambda: P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, scale=math.log(2.0), max_len=m)  # noqa: E731
    clean = call()
    assert bool(torch.isfinite(clean).all())
    for j in sorted({0, 1, 33, 64, top - 1, top + 1, top + 40, m // 2, m - 40, m - 1}):
        kept = pool.v.clone()
        put(pool, "v", 0, j, math.nan, d=7)
        got = call()
        want = torch.zeros_like(got, dtype=torch.bool)
        want[..., 7] = True
        assert torch.equal(torch.isnan(got), want) and torch.equal(got[~want], clean[~want]), j
        pool.v.copy_(kept)


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_sinks_of_any_size(P, codes):
    """A sink of +inf, or beyond what fp32 holds in base 2, takes all the weight, one of -inf or as far below none, one of NaN is NaN;
    as attention_prompt has it."""
    from tinygiant_b200 import attention as A
    g, H, hd = gen(55), 8, 64
    top = torch.finfo(torch.float32).max
    sinks = torch.tensor([math.inf, top, -math.inf, -top, math.nan, 0.5, 3e38, -3e38], device="cuda")
    for lens in ([40, 3, 0], [3000, 900, 0]):
        pool = Pool(g, torch.bfloat16, codes, H, hd, 16, lens)
        q = rand(g, 3, 1, H, hd, dtype=torch.bfloat16)
        got = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, sinks=sinks)
        plain = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw)
        assert not bool(got[:2, 0, [0, 1, 6]].any()) and torch.equal(got[:2, 0, [2, 3, 7]], plain[:2, 0, [2, 3, 7]])
        assert bool(torch.isnan(got[:2, 0, 4]).all()) and not bool(got[2].any())
        check(got[:2, :, 5], *(x[:2, :, 5] for x in paged_ref(pool, q, lens, 0, torch.full_like(sinks, 0.5))), codes)
        k, v = P.cache_gather(pool.k, pool.v, pool.tables, ends(lens), sum(lens), **pool.kw)
        prompt = A.attention_prompt(q[:, 0], k, v, ints(0, 1, 2, 3), ends(lens), sinks=sinks)
        assert torch.equal(torch.isnan(prompt[:2]), torch.isnan(got[:2, 0])) and not bool(prompt[:2, [0, 1, 6]].any())
