"""Attention over device tensors (tinygiant_b200.attention) against the
definitions in 64 bits: packed prompts, a shared prefix with gathered
weights, eviction; and what they refuse.

Tolerances, element by element.  u is the unit roundoff of the type (2^-8
bf16, 2^-11 fp16).  An output is rounded once (u |o|), the softmax weights may
be rounded to the type before their product with v (u A, A the weighted mean
of |v|), and each score is off by at most delta = (hd + 8) 2^-23 S, S the sum
of |scale q_d k_d| (fp32 sums, truncated or rounded, the scaling and the
exponential's 2^-22 and |x| 2^-23 included), which moves a weight by at most
2 delta of itself.  So |o - o64| <= u |o64| + (u + 2 delta) 1.05 A, and a
gathered weight is off by at most 2 delta w and the rounding of its sum."""
import ctypes
import math

import numpy as np
import pytest

import tinygiant_b200 as tg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def A(gpu):
    from tinygiant_b200 import attention
    return attention


def rand(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def attend(q, k, v, ok, scale, sink):
    """q [n, hd], k, v [m, hd], ok [n, m]: outputs, weights, A and delta, in 64 bits."""
    q, k = q.double(), k.double()
    x = torch.where(ok, q @ k.T * scale, -math.inf)
    s = torch.where(ok, q.abs() @ k.abs().T * abs(scale), 0.0)
    delta = (q.shape[1] + 8) * 2.0 ** -23 * (s.amax(1, keepdim=True) if s.shape[1] else s.new_zeros(len(q), 1))
    if sink is not None:
        x = torch.cat([x, torch.full((len(q), 1), float(sink), dtype=torch.float64, device=q.device)], 1)
    p = torch.nan_to_num(torch.softmax(x, 1), nan=0.0)[:, :k.shape[0]]
    v = torch.where(ok.any(0)[:, None], v.double(), 0.0)
    return p @ v, p, p @ v.abs(), delta


def check(got, want, a, delta):
    u = U[got.dtype]
    tol = u * want.abs() + (u + 2 * delta) * 1.05 * a + 2.0 ** -24
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))
    assert not bool(torch.isnan(got).any())


def ends(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def prompt_ref(q, k, v, nq, nk, window, sinks, scale):
    H, KH = q.shape[1], k.shape[1]
    out, a, delta = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(3))
    q0 = k0 = 0
    for n, m in zip(nq, nk):
        if n and m:
            i = torch.arange(n, device=q.device)[:, None] + (m - n)
            j = torch.arange(m, device=q.device)
            ok = (j <= i) & ((j > i - window) if window else torch.ones_like(j <= i))
            for h in range(H):
                kh = h // (H // KH)
                o, _, ah, d = attend(q[q0:q0 + n, h], k[k0:k0 + m, kh], v[k0:k0 + m, kh], ok, scale,
                                     None if sinks is None else sinks[h])
                out[q0:q0 + n, h], a[q0:q0 + n, h], delta[q0:q0 + n, h] = o, ah, d
        q0, k0 = q0 + n, k0 + m
    return out, a, delta


PROMPTS = [   # heads, kv heads, head_dim, queries, keys (None: as many), window, sinks
    (1, 1, 64, [1], None, 0, False),
    (8, 2, 64, [8], None, 0, True),
    (8, 1, 128, [127, 128, 129], None, 0, False),
    (4, 4, 128, [257, 1, 511], None, 0, False),
    (32, 4, 128, [0, 5, 0, 300, 0], None, 0, True),
    (14, 2, 64, [65, 19, 100], None, 0, False),
    (6, 2, 72, [33, 200], None, 0, False),
    (16, 1, 96, [40, 77], None, 0, True),
    (64, 1, 64, [37], None, 0, False),
    (128, 1, 128, [5, 3], None, 0, False),
    (5, 5, 8, [70, 3], None, 0, False),
    (9, 3, 40, [61], [190], 0, True),
    (8, 2, 128, [1, 1, 1], [1, 700, 2049], 0, False),
    (32, 4, 128, [8], [4096], 0, True),
    (8, 4, 64, [100, 16], [1000, 5000], 0, False),
    (8, 8, 64, [10, 7, 130], [4, 0, 129], 0, True),
    (8, 2, 64, [300, 40], None, 1, False),
    (8, 2, 64, [300, 40], None, 5, True),
    (16, 2, 64, [700, 129], None, 128, True),
    (8, 1, 128, [200, 50], [900, 3000], 300, False),
    (4, 2, 128, [600], None, 10000, False),
    (2, 1, 128, [1500], None, 0, False),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: "-".join(map(str, c[:3])) + f"-w{c[5]}-{sum(c[3])}")
def test_prompt_matches_definition(A, case, dtype):
    H, KH, hd, nq, nk, window, with_sinks = case
    g, dt = gen(1), DT[dtype]
    q = rand(g, sum(nq), H, hd, dtype=dt, scale=1.5)
    k, v = (rand(g, sum(nk or nq), KH, hd, dtype=dt) for _ in range(2))
    sinks = torch.randn(H, generator=g, device="cuda") if with_sinks else None
    got = A.attention_prompt(q, k, v, ends(nq), ends(nk) if nk else None, window=window, sinks=sinks,
                             max_k=max(nk or nq))
    check(got, *prompt_ref(q, k, v, nq, nk or nq, window, sinks, 1 / math.sqrt(hd)))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prompt_of_many_sequences(A, dtype):
    """More sequences than the plan holds at a time, and one long one among them that is split."""
    rng, g, dt, H, KH, hd = np.random.default_rng(41), gen(41), DT[dtype], 4, 2, 64
    nq = [int(n) for n in rng.integers(0, 6, 1500)]
    nk = [n + int(c) for n, c in zip(nq, rng.integers(0, 9, 1500))]
    nq[1200], nk[1200] = 3, 20000
    q = rand(g, sum(nq), H, hd, dtype=dt, scale=1.5)
    k, v = (rand(g, sum(nk), KH, hd, dtype=dt) for _ in range(2))
    got = A.attention_prompt(q, k, v, ends(nq), ends(nk), max_k=20000)
    check(got, *prompt_ref(q, k, v, nq, nk, 0, None, 1 / 8))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prompt_strided_views(A, dtype):
    """Views of one fused q/k/v tensor, of head-major tensors, and a strided output."""
    g, dt, H, KH, hd, nq = gen(2), DT[dtype], 8, 2, 64, [150, 33]
    T = sum(nq)
    fused = rand(g, T, H + 2 * KH, hd, dtype=dt)
    q, k, v = fused[:, :H], fused[:, H:H + KH], fused[:, H + KH:]
    want = prompt_ref(q, k, v, nq, nq, 0, None, 0.25)
    check(A.attention_prompt(q, k, v, ends(nq), scale=0.25), *want)
    qh, kh, vh = (x.permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in (q, k, v))
    wide = torch.full((T, H, hd + 8), 7.0, dtype=dt, device="cuda")
    got = A.attention_prompt(qh, kh, vh, ends(nq), scale=0.25, out=wide[..., :hd])
    check(got, *want)
    assert bool((wide[..., hd:] == 7.0).all())


def test_prompt_large_scores_and_sinks(A):
    """Scores of hundreds: nearly one-hot softmax; sinks far above and far below them, and -inf."""
    g, H, KH, hd, nq = gen(3), 8, 4, 128, [260]
    q, k, v = rand(g, 260, H, hd, dtype=torch.float16, scale=20), *(rand(g, 260, KH, hd, dtype=torch.float16, scale=s) for s in (10, 1))
    sinks = torch.tensor([0.0, 1e4, -1e4, -math.inf, 50.0, 300.0, -math.inf, 0.0], device="cuda")
    got = A.attention_prompt(q, k, v, ends(nq), sinks=sinks)
    check(got, *prompt_ref(q, k, v, nq, nq, 0, sinks, 1 / math.sqrt(hd)))


def test_prompt_rising_scores(A):
    """Scores that rise along the keys, so the running maximum moves in every tile, and that fall."""
    hd, n = 64, 1100
    up = torch.linspace(0, 60, n, device="cuda")
    for ramp in (up, up.flip(0)):
        k = torch.zeros(n, 1, hd, device="cuda")
        k[:, 0, 0] = ramp
        k, q = k.to(torch.bfloat16), torch.zeros(n, 2, hd, dtype=torch.bfloat16, device="cuda")
        q[:, :, 0] = 8
        v = rand(gen(4), n, 1, hd, dtype=torch.bfloat16)
        check(A.attention_prompt(q, k, v, ends([n])), *prompt_ref(q, k, v, [n], [n], 0, None, 1 / 8))


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_prompt_sequences_do_not_touch(A, poison):
    """A neighbour's keys and values that are not finite leave a sequence's outputs as they are."""
    g, H, KH, hd, nq = gen(5), 8, 2, 64, [70, 90, 200]
    T = sum(nq)
    q, k, v = rand(g, T, H, hd, dtype=torch.bfloat16), *(rand(g, T, KH, hd, dtype=torch.bfloat16) for _ in range(2))
    clean = A.attention_prompt(q, k, v, ends(nq))
    k[70:160], v[70:160] = poison, poison
    got = A.attention_prompt(q, k, v, ends(nq))
    assert torch.equal(got[:70], clean[:70]) and torch.equal(got[160:], clean[160:])


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("H,KH,hd,nq,nk,window", [(8, 2, 64, [300, 40], None, 0), (2, 2, 128, [500], None, 100),
                                                  (8, 1, 128, [8, 3], [3000, 260], 0), (4, 4, 96, [260], [700], 150)])
def test_prompt_values_do_not_reach_rows_that_do_not_see_them(A, H, KH, hd, nq, nk, window, poison):
    """A value row that is not finite changes the rows that attend to its key and no other; those get it in its dimension."""
    g, dt = gen(32), torch.bfloat16
    nk = nk or nq
    q, k, v = rand(g, sum(nq), H, hd, dtype=dt), *(rand(g, sum(nk), KH, hd, dtype=dt) for _ in range(2))
    run = lambda: A.attention_prompt(q, k, v, ends(nq), ends(nk), window=window)  # noqa: E731
    clean = run()
    n, m = nq[0], nk[0]
    at = [m - 1, m - 2 if n > 2 else m - 1, max(0, m - n + n // 2)]      # the last keys and one amid the queries
    dim = [3, hd - 1, 0]
    for j, d in zip(at, dim):
        v[j, KH - 1, d] = poison
    got = run()
    want = clean.clone()
    i = torch.arange(n, device="cuda") + (m - n)
    for j, d in zip(at, dim):
        sees = (i >= j) & ((i - j < window) if window else True)
        heads = range(H - H // KH, H)
        for h in heads:
            want[:n, h, d] = torch.where(sees, torch.tensor(poison, dtype=dt, device="cuda"), want[:n, h, d])
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    # a weight that is 0 in the type makes a NaN of an infinity: rows that see the key may have that instead
    same |= torch.isnan(got) & torch.isinf(want)
    assert bool(same.all()), int((~same).sum())


def test_shared_prefix_values_outside_the_window(A):
    """A prefix value that is not finite, before the window of some sequences: those do not see it."""
    g, dt, H, KH, hd, P = gen(33), torch.bfloat16, 8, 2, 64, 300
    q = rand(g, 3, H, hd, dtype=dt)
    pk, pv = (rand(g, KH, P, hd, dtype=dt) for _ in range(2))
    k, v = (rand(g, 3, KH, 64, hd, dtype=dt) for _ in range(2))
    n = torch.tensor([60, 5, 55], dtype=torch.int32, device="cuda")
    run = lambda: A.attention_shared(q, pk, pv, k, v, n, window=100)  # noqa: E731
    clean = run()
    pv[:, 250, 7] = math.inf            # seen from position 304 (back to 205), not from 359 (260) and 354 (255)
    got = run()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    assert bool(torch.isinf(got[1, :, 7]).all()) and torch.equal(got[1, :, :7], clean[1, :, :7])


def test_prompt_on_another_stream_and_in_a_graph(A):
    g, nq = gen(6), [100, 28]
    q, k, v = rand(g, 128, 8, 64, dtype=torch.bfloat16), *(rand(g, 128, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    cu = ends(nq)
    want = A.attention_prompt(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = A.attention_prompt(q, k, v, cu)
    s.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.attention_prompt(q, k, v, cu, out=out)
    q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, A.attention_prompt(q, k, v, cu))


def test_prompt_twice_gives_the_same_bits(A):
    g, nq, nk = gen(7), [9, 700], [3000, 900]
    q, k, v = rand(g, 709, 8, 128, dtype=torch.bfloat16), *(rand(g, 3900, 1, 128, dtype=torch.bfloat16) for _ in range(2))
    outs = [A.attention_prompt(q, k, v, ends(nq), ends(nk)) for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_empty_calls(A):
    """No rows, no keys, no sequences: nothing, or zeros."""
    bf = torch.bfloat16
    q, k = torch.ones(6, 4, 64, dtype=bf, device="cuda"), torch.ones(0, 2, 64, dtype=bf, device="cuda")
    assert A.attention_prompt(q[:0], k, k, ends([0]), ends([0])).shape == (0, 4, 64)
    assert not bool(A.attention_prompt(q, k, k, ends([4, 2]), ends([0, 0])).any())
    c, n = torch.ones(6, 2, 0, 64, dtype=bf, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    w = torch.zeros(6, 2, 0, device="cuda")
    assert not bool(A.attention_shared(q, None, None, c, c, n, weights=w).any())
    assert A.attention_shared(q[:0], None, None, c[:0], c[:0], n[:0]).shape == (0, 4, 64)
    p = torch.ones(2, 3, 64, dtype=bf, device="cuda")
    assert bool((A.attention_shared(q, p, p, c, c, n) == 1).all())      # the prefix alone: the mean of ones


def test_prompt_offsets_past_the_rows_stay_inside(A):
    """Offsets beyond the tensors read as their ends: no access outside, other sequences unharmed."""
    g = gen(8)
    q, k, v = rand(g, 64, 4, 64, dtype=torch.bfloat16), *(rand(g, 64, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    cu = torch.tensor([0, 40, 64], dtype=torch.int32, device="cuda")
    far = torch.tensor([0, 40, 1 << 30], dtype=torch.int32, device="cuda")
    want = A.attention_prompt(q, k, v, cu)
    got = A.attention_prompt(q, k, v, far, far)
    assert torch.equal(got[:40], want[:40])
    torch.cuda.synchronize()


def shared_ref(q, pk, pv, k, v, lens, window, sinks, scale):
    (B, H, hd), KH = q.shape, k.shape[1]
    P = 0 if pk is None else pk.shape[1]
    out, a = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    delta = torch.zeros(B, H, 1, dtype=torch.float64, device=q.device)
    w, wd = (torch.zeros(k.shape[:3], dtype=torch.float64, device=q.device) for _ in range(2))
    for b, n in enumerate(lens):
        for h in range(H):
            kh = h // (H // KH)
            kk = k[b, kh, :n] if P == 0 else torch.cat([pk[kh], k[b, kh, :n]])
            vv = v[b, kh, :n] if P == 0 else torch.cat([pv[kh], v[b, kh, :n]])
            if len(kk) == 0:
                continue
            j = torch.arange(P + n, device=q.device)
            ok = (j >= P + n - window if window else j >= 0)[None]
            o, p, ah, d = attend(q[b, h][None], kk, vv, ok, scale, None if sinks is None else sinks[h])
            out[b, h], a[b, h], delta[b, h] = o[0], ah[0], d[0]
            w[b, kh, :n] += p[0, P:]
            wd[b, kh, :n] += 2 * d[0] * p[0, P:]
    return out, a, delta, w, wd


SHARED = [    # heads, kv heads, head_dim, prefix, cap, lens, window, sinks
    (1, 1, 64, 0, 8, [1], 0, False),
    (8, 2, 64, 1, 8, [0, 1, 8], 0, True),
    (32, 4, 128, 100, 64, [17, 33], 0, False),
    (32, 4, 128, 0, 300, [300, 0, 129, 64], 0, True),
    (8, 1, 128, 129, 1, [1] * 40, 0, False),
    (8, 2, 64, 1000, 600, [600, 0, 1, 31, 513, 256, 257], 0, False),
    (14, 2, 96, 333, 77, [77, 5, 60], 0, False),
    (6, 2, 40, 64, 200, [199, 65], 0, True),
    (16, 1, 64, 300, 130, [130] * 19, 0, False),
    (48, 2, 128, 200, 90, [90, 33, 1], 0, True),
    (128, 1, 64, 40, 90, [90, 33], 0, False),
    (5, 5, 8, 70, 33, [33, 2], 0, False),
    (8, 2, 64, 500, 300, [300, 3, 100, 0], 64, False),
    (8, 2, 128, 900, 200, [200, 3, 100, 0, 150], 400, True),
    (8, 4, 128, 50, 40, [40, 10], 100000, False),
    (8, 2, 64, 200, 100, [50, 7], 1, False),
    (32, 4, 128, 5000, 2000, [2000, 1111], 0, False),
    (8, 1, 128, 0, 9000, [9000], 0, True),
    (4, 2, 64, 40, 300, [(i * 37) % 301 for i in range(300)], 0, False),     # more sequences than a scan takes at once
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", SHARED, ids=lambda c: "-".join(map(str, c[:5])) + f"-w{c[6]}")
def test_shared_matches_definition(A, case, dtype):
    """Outputs and weights; the rows behind each sequence's end hold NaN."""
    H, KH, hd, P, cap, lens, window, with_sinks = case
    g, dt, B = gen(11), DT[dtype], len(lens)
    q = rand(g, B, H, hd, dtype=dt, scale=1.5)
    pk, pv = (rand(g, KH, P, hd, dtype=dt) if P else None for _ in range(2))
    k, v = (rand(g, B, KH, cap, hd, dtype=dt) for _ in range(2))
    for b, n in enumerate(lens):
        k[b, :, n:], v[b, :, n:] = math.nan, math.nan
    sinks = torch.randn(H, generator=g, device="cuda") if with_sinks else None
    w0 = torch.rand(B, KH, cap, generator=g, device="cuda")
    w = w0.clone()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = A.attention_shared(q, pk, pv, k, v, n, window=window, sinks=sinks, weights=w)
    out, a, delta, ww, wd = shared_ref(q, pk, pv, k, v, lens, window, sinks, 1 / math.sqrt(hd))
    check(got, out, a, delta)
    tol = 1.05 * wd + (ww + w0) * 2.0 ** -22
    assert bool(((w.double() - w0 - ww).abs() <= tol).all()), float(((w.double() - w0 - ww).abs() / tol).max())
    assert torch.equal(A.attention_shared(q, pk, pv, k, v, n, window=window, sinks=sinks, max_len=max(lens)), got)


def test_shared_equals_a_prompt_of_its_last_row(A):
    """The same attention through the other operator: each sequence's keys laid out whole."""
    g, H, KH, hd, P, lens = gen(12), 8, 2, 128, 260, [5, 0, 130]
    q = rand(g, 3, H, hd, dtype=torch.float16)
    pk, pv = (rand(g, KH, P, hd, dtype=torch.float16) for _ in range(2))
    k, v = (rand(g, 3, KH, 130, hd, dtype=torch.float16) for _ in range(2))
    got = A.attention_shared(q, pk, pv, k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    whole = lambda p, x: torch.cat([torch.cat([p, x[b, :, :n]], 1).transpose(0, 1) for b, n in enumerate(lens)])  # noqa: E731
    want = A.attention_prompt(q, whole(pk, k), whole(pv, v), ends([1, 1, 1]), ends([P + n for n in lens]))
    assert float((got.double() - want.double()).abs().max()) <= 4 * U[torch.float16] * float(v.abs().max())


def test_shared_views_and_long_strides(A):
    """Caches as views of a position-major tensor; sequences more than 2^31 elements apart."""
    g, H, KH, hd, cap, lens = gen(13), 8, 2, 64, 96, [96, 50]
    kv = rand(g, 2, cap, 2 * KH, hd, dtype=torch.bfloat16)
    k, v = kv[:, :, :KH].transpose(1, 2), kv[:, :, KH:].transpose(1, 2)
    pre = rand(g, 40, 2 * KH, hd, dtype=torch.bfloat16)
    pk, pv = pre[:, :KH].transpose(0, 1), pre[:, KH:].transpose(0, 1)
    qq = rand(g, 2, 2 * H, hd, dtype=torch.bfloat16)
    q, n = qq[:, H:], torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, a, delta, ww, wd = shared_ref(q, pk, pv, k, v, lens, 0, None, 1 / 8)
    check(A.attention_shared(q, pk, pv, k, v, n), out, a, delta)
    apart = (1 << 31) + 64
    big = torch.zeros(apart + KH * cap * hd, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(big, (2, KH, cap, hd), (apart, cap * hd, hd, 1))
    far.copy_(k)
    w = torch.zeros(2, KH, 2 * cap, device="cuda")[:, :, :cap]
    got = A.attention_shared(q, pk, pv, far, v, n, weights=w)
    check(got, out, a, delta)
    assert bool(((w.double() - ww).abs() <= 1.05 * wd + ww * 2.0 ** -22).all())
    ko, _, wo, _, idx = A.cache_evict(far, v, w, n, 40, 8)
    at = idx.long()[..., None].expand(2, KH, 40, hd)
    assert torch.equal(ko, torch.gather(k, 2, at)) and torch.equal(wo, torch.gather(w, 2, idx.long()))


def test_shared_lengths_outside_their_range(A):
    g = gen(14)
    q = rand(g, 3, 4, 64, dtype=torch.bfloat16)
    k, v = (rand(g, 3, 2, 32, 64, dtype=torch.bfloat16) for _ in range(2))
    n = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = A.attention_shared(q, None, None, k, v, n(-5, 1 << 30, 20), max_len=20)
    assert torch.equal(got, A.attention_shared(q, None, None, k, v, n(0, 20, 20)))
    assert not bool(got[0].any())


def test_shared_twice_gives_the_same_bits(A):
    g, lens = gen(15), [700, 3, 0, 512, 129] * 8
    q = rand(g, 40, 32, 128, dtype=torch.bfloat16)
    pk, pv = (rand(g, 4, 1000, 128, dtype=torch.bfloat16) for _ in range(2))
    k, v = (rand(g, 40, 4, 700, 128, dtype=torch.bfloat16) for _ in range(2))
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    both = []
    for _ in range(2):
        w = torch.zeros(40, 4, 700, device="cuda")
        both.append((A.attention_shared(q, pk, pv, k, v, n, weights=w), w))
    assert torch.equal(both[0][0], both[1][0]) and torch.equal(both[0][1], both[1][1])


def evict_ref(w, lens, keep, recent):
    """Old positions that stay, [B, KH, keep], -1 behind the end."""
    B, KH, _ = w.shape
    idx = np.full((B, KH, keep), -1, np.int32)
    for b, n in enumerate(lens):
        m = min(n, keep)
        r = min(recent, m)
        for h in range(KH):
            x = w[b, h, :n - r].astype(np.float64)
            x = np.where(np.isnan(x), np.inf, x)
            more = np.isnan(w[b, h, :n - r])
            heavy = np.lexsort((np.arange(n - r), -x, ~more))[:m - r]
            idx[b, h, :m] = np.concatenate([np.sort(heavy), np.arange(n - r, n)])
    return idx


EVICT = [     # kv heads, head_dim, cap, lens, keep, recent
    (1, 64, 1, [1, 0], 1, 0),
    (2, 8, 10, [10, 3, 0, 7], 4, 2),
    (4, 128, 300, [300, 257], 256, 32),
    (2, 128, 1000, [1000, 999, 513, 512, 511], 512, 0),
    (3, 72, 700, [700, 650, 20], 100, 100),
    (2, 64, 700, [700, 650, 20], 700, 5),
    (1, 40, 5000, [5000, 4097], 1, 1),
    (1, 96, 5000, [5000, 4097], 1, 0),
    (2, 64, 40000, [40000, 33333], 10001, 77),
    (1, 8, 50000, [50000, 41000], 20000, 300),     # more weights than shared memory holds
]


@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(map(str, c[:3])) + f"-{c[4]}-{c[5]}")
def test_evict_matches_definition(A, case, kind):
    KH, hd, cap, lens, keep, recent = case
    rng, B = np.random.default_rng(21), len(case[3])
    w = np.exp(1.5 * rng.standard_normal((B, KH, cap))).astype(np.float32)
    if kind == "ties":
        w = np.floor(w * 2) / 2                 # few values, many of them zero
    if kind == "special":
        odd = np.array([np.nan, np.inf, -np.inf, -0.0, 0.0, -1.5, 1e-42, -np.nan], np.float32)
        w = np.where(rng.random(w.shape) < 0.5, odd[rng.integers(0, len(odd), w.shape)], w)
    g = gen(22)
    k, v = rand(g, B, KH, cap, hd, dtype=torch.bfloat16), rand(g, B, KH, cap, hd, dtype=torch.bfloat16)
    wt = torch.from_numpy(w).cuda()
    ko, vo, wo, lo, idx = A.cache_evict(k, v, wt, torch.tensor(lens, dtype=torch.int32, device="cuda"), keep, recent)
    want = evict_ref(w, lens, keep, recent)
    assert np.array_equal(idx.cpu().numpy(), want)
    assert lo.tolist() == [min(n, keep) for n in lens]
    at = torch.from_numpy(want).cuda().long()
    gone = at < 0
    rows = at.clamp(min=0)[..., None].expand(B, KH, keep, hd)
    assert torch.equal(ko, torch.gather(k, 2, rows).masked_fill(gone[..., None], 0))
    assert torch.equal(vo, torch.gather(v, 2, rows).masked_fill(gone[..., None], 0))
    assert torch.equal(wo.view(torch.int32), torch.gather(wt, 2, rows[..., 0]).masked_fill(gone, 0).view(torch.int32))


def test_evict_views_and_an_empty_batch(A):
    g, KH, hd, cap = gen(23), 2, 64, 50
    kv = rand(g, 3, cap, 2 * KH, hd, dtype=torch.float16)
    k, v = kv[:, :, :KH].transpose(1, 2), kv[:, :, KH:].transpose(1, 2)
    w = torch.rand(3, KH, 2 * cap, generator=g, device="cuda")[:, :, :cap]
    n = torch.tensor([50, 30, 99], dtype=torch.int32, device="cuda")      # 99: counts as 50
    got = A.cache_evict(k, v, w, n, 20, 4)
    want = A.cache_evict(k.contiguous(), v.contiguous(), w.contiguous(), n.clamp(max=50), 20, 4)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert A.cache_evict(k[:0], v[:0], w[:0], n[:0], 20, 4)[0].shape == (0, KH, 20, hd)


def test_a_sequence_decodes_through_an_eviction(A):
    """Prompt, tokens with gathered weights, eviction, one more token: each step against the definition."""
    g, H, KH, hd, T, cap = gen(24), 8, 2, 64, 90, 100
    dt = torch.bfloat16
    k, v = (torch.zeros(1, KH, cap, hd, dtype=dt, device="cuda") for _ in range(2))
    q, kp, vp = rand(g, T, H, hd, dtype=dt), rand(g, T, KH, hd, dtype=dt), rand(g, T, KH, hd, dtype=dt)
    check(A.attention_prompt(q, kp, vp, ends([T])), *prompt_ref(q, kp, vp, [T], [T], 0, None, 1 / 8))
    k[0, :, :T], v[0, :, :T] = kp.transpose(0, 1), vp.transpose(0, 1)
    w, n = torch.zeros(1, KH, cap, device="cuda"), T
    want = torch.zeros(1, KH, cap, dtype=torch.float64, device="cuda")
    for _ in range(10):
        k[0, :, n], v[0, :, n] = rand(g, KH, hd, dtype=dt), rand(g, KH, hd, dtype=dt)
        n += 1
        qt = rand(g, 1, H, hd, dtype=dt)
        got = A.attention_shared(qt, None, None, k, v, torch.tensor([n], dtype=torch.int32, device="cuda"), weights=w)
        out, a, delta, ww, _ = shared_ref(qt, None, None, k, v, [n], 0, None, 1 / 8)
        check(got, out, a, delta)
        want += ww
    assert float((w.double() - want).abs().max()) < 1e-4
    k2, v2, w2, n2, idx = A.cache_evict(k, v, w, torch.tensor([n], dtype=torch.int32, device="cuda"), 40, 10)
    assert np.array_equal(idx.cpu().numpy(), evict_ref(w.cpu().numpy(), [n], 40, 10)) and n2.tolist() == [40]
    qt = rand(g, 1, H, hd, dtype=dt)
    out, a, delta, _, _ = shared_ref(qt, None, None, k2, v2, [40], 0, None, 1 / 8)
    check(A.attention_shared(qt, None, None, k2, v2, n2, weights=w2), out, a, delta)


def test_refusals(A):
    """What the Python entries refuse, before anything runs."""
    bf, cu = torch.bfloat16, ends([4])
    q, k = torch.zeros(4, 4, 64, dtype=bf, device="cuda"), torch.zeros(4, 2, 64, dtype=bf, device="cuda")

    def no(text, fn, *args, **kw):
        with pytest.raises(ValueError, match=text):
            fn(*args, **kw)

    P = A.attention_prompt
    no("CUDA tensor", P, q.cpu(), k, k, cu)
    no("bfloat16 or float16", P, q.float(), k, k, cu)
    no("all of one type", P, q, k.half(), k, cu)
    no("3 dimensions", P, q[0], k, k, cu)
    no("do not share", P, q[:, :3], k, k, cu)
    no("multiple of 8", P, q[..., :60], k[..., :60], k[..., :60], cu)
    no("at most 128", P, *(torch.zeros(4, 2, 136, dtype=bf, device="cuda") for _ in range(3)), cu)
    no("do not fit", P, q, k, k[:, :, :32], cu)
    no("strides", P, torch.zeros(4, 4, 68, dtype=bf, device="cuda")[..., :64], k, k, cu)
    no("strides", P, q, k[:, :1].expand(4, 2, 64), k, cu)
    no("contiguous", P, q, k.transpose(1, 2).contiguous().transpose(1, 2), k, cu)
    no("cu_q", P, q, k, k, cu.long())
    no("cu_k", P, q, k, k, cu, ends([2, 2]))
    no("as many keys", P, q, k[:3], k[:3], cu)
    no("sinks", P, q, k, k, cu, sinks=torch.zeros(2, device="cuda"))
    no("window", P, q, k, k, cu, window=-1)
    no("shape of q", P, q, k, k, cu, out=torch.zeros(4, 2, 64, dtype=bf, device="cuda"))
    with pytest.raises(tg.TinyGiantCudaError, match="aligned"):
        P(torch.zeros(4 * 4 * 64 + 4, dtype=bf, device="cuda")[4:].view(4, 4, 64), k, k, cu)
    for scale in (math.nan, math.inf, 0.0, -1.0):
        with pytest.raises(tg.TinyGiantCudaError, match="scale"):
            P(q, k, k, cu, scale=scale)
    S, c, n = A.attention_shared, torch.zeros(4, 2, 8, 64, dtype=bf, device="cuda"), ends([1] * 3)
    no("do not fit", S, q, None, None, c[:3], c[:3], n)
    no("prefix_k and prefix_v", S, q, k.transpose(0, 1), None, c, c, n)
    no("prefix_k and prefix_v", S, q, k.transpose(0, 1)[:1], k.transpose(0, 1)[:1], c, c, n)
    no("lens", S, q, None, None, c, c, n[:3])
    no("weights", S, q, None, None, c, c, n, weights=torch.zeros(4, 2, 8, dtype=bf, device="cuda"))
    no("broadcast", S, q, None, None, c, c, n, weights=torch.zeros(1, 2, 8, device="cuda").expand(4, 2, 8))
    no("max_len", S, q, None, None, c, c, n, max_len=-1)
    E, w = A.cache_evict, torch.zeros(4, 2, 8, device="cuda")
    no("need 0 < keep", E, c, c, w, n, 0, 0)
    no("need 0 < keep", E, c, c, w, n, 9, 0)
    no("need 0 < keep", E, c, c, w, n, 4, 5)
    no("weights", E, c, c, w[:, :1], n, 4, 1)
    no("one shape", E, c, c[:, :, :7], w, n, 4, 1)
    assert not bool(P(q, k, k, cu).any())      # and the next good call runs


def test_no_device_error_is_pending(A, gpu):
    """tg_cuda_synchronize reports the operators' device errors; good calls leave none."""
    g = gen(31)
    q, k, v = rand(g, 300, 8, 128, dtype=torch.bfloat16), *(rand(g, 300, 2, 128, dtype=torch.bfloat16) for _ in range(2))
    A.attention_prompt(q, k, v, ends([300]))
    torch.cuda.synchronize()
    assert gpu.tg_cuda_synchronize() == 0, tg.last_error(gpu)


def test_c_entries_refuse_host_memory(gpu):
    """Pointers to host memory, small workspaces and overlapping outputs, at the C entries."""
    lib, h = gpu, np.zeros(4096, np.float32)
    d = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda").data_ptr()
    cu = ends([4]).data_ptr()
    st = (ctypes.c_int64 * 16)(*[64] * 16)
    args = lambda q, out: (0, q, d, d, out, cu, cu, None, 1, 4, 4, 4, 1, 1, 64, st, 0, 0.125, None, 0, None)  # noqa: E731
    assert lib.tg_attention_prompt(*args(h.ctypes.data, d)) == 3 and "device memory" in tg.last_error(lib)[1]
    assert lib.tg_attention_prompt(*args(d, None)) == 3 and "device memory" in tg.last_error(lib)[1]
    rc = lib.tg_cache_evict(d, d, d, d, d, d + 4096, d + 8192, d + 12288, d + 16384, 1, 8, 1, 64, st, 4, 1, None)
    assert rc == 3 and "overlap" in tg.last_error(lib)[1]


def test_serving_example(gpu):
    """Prompts, decoding, evictions and the experts' steps through examples/serve_batch.py, the last attention checked."""
    import importlib.util
    from pathlib import Path
    spec = importlib.util.spec_from_file_location("serve_batch", Path(__file__).resolve().parents[1] / "examples" / "serve_batch.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(["--batch", "5", "--prefix", "130", "--steps", "30", "--cap", "130", "--keep", "100", "--recent", "20"]) < 2e-2
