"""The paged cache where it can go wrong: values that are not finite beside cuts, codes and scales next to a border,
earlier scales of any kind, the C entries by their argument lists, and what is refused beside the ordinary.

Tolerances: none, but where a test derives its own.  Codes, scales and NaN are compared for equality; expected codes are worked out on the host in
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


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("m", [7, 60, 3000])
def test_weights_keep_more_bits_than_the_values(P, m, codes, dtype):
    """Three keys of weight 1 and values of 1 against four of weight r and -1, r = 0.75 and 2^-12.2 (bf16 pages: 2^-9.2) more, which one
    fp16 (or bf16) weight would round to 0.75: the output is what that drops.

    Tolerance: u |o| for the output, and of A = 1 at most the weights' 2^-22 (2^-16), twice delta = (hd + 16) 2^-23 S + 2^-18 with S = scale
    < 0.3, and fp32's sums."""
    g, dt, hd = gen(56), DT[dtype], 16
    pool = Pool(g, dt, codes, 1, hd, 16, [m])
    for x, fill in (("k", -448.0), ("v", 0.0)):                     # the other keys' weights are e^-128
        pages = getattr(pool, x)
        pages.copy_(torch.full(pages.shape, fill, device="cuda").to(pages.dtype))
        if codes:
            getattr(pool, x + "s").fill_(1.0)
    at = [round(i * (m - 1) / 6) for i in range(7)]
    for i, j in enumerate(at):
        put(pool, "k", 0, j, -1.0 if i % 2 == 0 else 0.0)
        put(pool, "v", 0, j, -1.0 if i % 2 == 0 else 1.0)
    q = torch.zeros(1, 1, 3, hd, dtype=dt, device="cuda")
    q[..., 0] = 1.0
    one, w = (2.0 ** -9.2, 2.0 ** -16) if dtype == "bf16" and not codes else (2.0 ** -12.2, 2.0 ** -22)
    for more in (one, -one):
        scale = float(np.float32(-math.log(0.75 * (1 + more))))
        r = math.exp(-scale)
        want = (3 - 4 * r) / (3 + 4 * r)
        got = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, scale=scale, max_len=m).double()
        u = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
        tol = u * abs(want) + w + 2 * (32 * 2.0 ** -23 * scale + 2.0 ** -18)
        assert abs(want) > 4 * tol and bool(((got - want).abs() <= tol).all()), (got[0, 0, 0, 0].item(), want)


@pytest.mark.parametrize("power", [-110, -20, 0, 20, 97])
def test_queries_of_a_wide_range_over_codes(P, power):
    """bf16 queries one value of which is 2^30 times the others and meets keys of zero: the others keep all their bits."""
    g, m, hd = gen(57), 300, 64
    pool = Pool(g, torch.bfloat16, True, 1, hd, 16, [m])
    k = pool.k.float()
    k[..., 9] = 0.0
    pool.k.copy_(k.to(E4M3))
    q = rand(g, 1, 1, 8, hd, dtype=torch.bfloat16).abs().clamp(0.51, 0.99)
    q[..., 9] = 2.0 ** 30
    scale = 2.0 ** -power / 8
    q = (q.float() * 2.0 ** power).to(torch.bfloat16)
    got = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, scale=scale)
    check(got, *paged_ref(pool, q, [m], scale=scale), True)


# ---- codes next to a border

E4M3_VALUES = np.array([0.0, *(m / 512 for m in range(1, 8)), *((8 + m) / 8 * 2.0 ** e for e in range(-6, 9) for m in range(8))][:127], dtype=L)


def nearest(y):
    """The nearest values of e4m3 of long doubles, |y| <= 448, none a tie."""
    y = np.asarray(y, dtype=L)
    d = np.abs(np.abs(y)[..., None] - E4M3_VALUES)
    i = d.argmin(-1)
    two = np.partition(d, 1, axis=-1)
    assert bool((two[..., 1] - two[..., 0] > np.abs(y) * L(2) ** -44).all()), "an input of this test is too near a tie"
    return np.sign(y) * E4M3_VALUES[i]


def border(y):
    """The border between two codes that is nearest to y > 0, in [16, 448)."""
    step = 2.0 ** (math.floor(math.log2(y)) - 3)
    return (math.floor(y / step) + 0.5) * step


def bf16(rng, low, high, n):
    x = torch.from_numpy(rng.uniform(low, high, n)).to(torch.bfloat16)
    return x, x.double().numpy()


def one_token(P, rows, freqs, position=None, ctx=0, before=None, **kw):
    """One token of one sequence (rows [KH, hd] bf16: key and value) after ctx others, in pages of 8 bits: its codes of K as numbers,
    and the scales of K and V [KH].  before: the block's scales there."""
    KH, hd = rows.shape
    k_pages, v_pages = (torch.zeros(1, KH, 16, hd, device="cuda").to(E4M3) for _ in range(2))
    ks, vs = (torch.full((1, KH, 1), 1.0, device="cuda") if before is None else before.clone().view(1, KH, 1) for _ in range(2))
    x = rows.cuda()[None]
    P.cache_append(x, x, k_pages, v_pages, ints(0).view(1, 1), ints(ctx + 1), k_scales=ks, v_scales=vs,
                   freqs=None if freqs is None else torch.from_numpy(freqs).cuda(), positions=None if position is None else ints(position), **kw)
    f = lambda t: t[0, :, ctx].float().cpu().numpy().astype(L)  # noqa: E731
    return f(k_pages), f(v_pages), ks[0, :, 0].cpu().numpy().astype(L), vs[0, :, 0].cpu().numpy().astype(L)


def turned(a, b, p, f):
    with decimal.localcontext(decimal.Context(prec=60)):
        around = decimal.Decimal("6.28318530717958647692528676655900576839433879875021164")
        t = np.array([L(str(decimal.Decimal(p) * decimal.Decimal(float(x)) % around)) for x in f], dtype=L)
    c, s = np.cos(t), np.sin(t)
    return a * c - b * s, b * c + a * s


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("p,low,high", [(1, 0.70, 0.7853), (1, 0.0, 6.28), (1048573, 0.0, 6.28), (2000003, 0.0, 6.28)])
def test_codes_of_angles_next_to_a_border(P, p, low, high, interleaved):
    """Frequencies that take a pair's first value to a border between two codes, 2^-32 of it to either side (at far positions as near
    as a frequency in fp64 gets)."""
    rng, n = np.random.default_rng(61 + p), 32
    for _ in range(12):
        a, b, f = np.zeros(n), np.zeros(n), np.zeros(n)
        a[0] = 300.0                                               # the scale is 1
        for j in range(1, n):
            while True:
                (_, x), (_, y) = bf16(rng, -250, 250, 1), bf16(rng, -250, 250, 1)
                r, phi, t0 = np.sqrt(L(x[0]) ** 2 + L(y[0]) ** 2), np.arctan2(L(y[0]), L(x[0])), rng.uniform(low, high)
                y0 = float(r) * math.cos(t0 + float(phi))
                if not 20 < abs(y0) < 0.9 * float(r):
                    continue
                aim = L(border(abs(y0)) * math.copysign(1, y0)) * (1 + L(2) ** -32 * (1 if rng.random() < 0.5 else -1))
                for theta in (np.arccos(aim / r), -np.arccos(aim / r)):
                    t = theta - phi
                    t += L("6.28318530717958647692528676655900577") * np.round((t0 - t) / (L("6.28318530717958647692528676655900577")))
                    if abs(t - t0) < 0.1 and low <= t <= high:
                        break
                else:
                    continue
                # a far position: as many whole turns more as make the frequency one of 0.5 to 1
                turns = 0 if p == 1 else int(rng.uniform(0.5, 1) * p / 6.3)
                f[j] = np.float64((t + turns * L("6.28318530717958647692528676655900577")) / p)
                ya, yb = turned(L(x[0]), L(y[0]), p, f[j:j + 1])
                near_tie = min(abs(abs(v) / L(border(float(abs(v)))) - 1) if abs(v) >= 16 else 1 for v in (ya[0], yb[0]))
                if near_tie > L(2) ** -41 and abs(yb[0]) > 16:
                    a[j], b[j] = x[0], y[0]
                    break
        ya, yb = turned(a.astype(L), b.astype(L), p, f)
        row = np.empty(2 * n)
        want = np.empty(2 * n, dtype=L)
        lo, hi = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, n), slice(n, None))
        row[lo], row[hi], want[lo], want[hi] = a, b, nearest(ya), nearest(yb)
        got, _, ks, _ = one_token(P, torch.from_numpy(row).to(torch.bfloat16)[None], f, position=p, interleaved=interleaved)
        assert ks[0] == 1 and np.array_equal(got[0], want), int((got[0] != want).sum())


@pytest.mark.parametrize("f", [0.7, 1e3, 1.7e7, 1.3e9, 2.1e12, 1e18, 1e40])
def test_frequencies_of_any_size(P, f):
    """Angles of more turns than fp64 counts: to 2^-20 as long as a position's turns are below 2^60, and a rotation always."""
    pos = ints(0, 1, -1, 77777, 123456789, -987654321, 2147483647, -2147483647)
    freqs = torch.tensor([f * 2.0 ** -i for i in range(32)], dtype=torch.float64, device="cuda")
    q = torch.zeros(8, 1, 64, dtype=torch.float16, device="cuda")
    q[..., :32] = 1.0
    got = P.rotary(q, None, pos, freqs)[0][:, 0].double()
    # fp16 rounds by 2^-11 at most, fp32's sine and cosine by 2^-25, twice
    assert bool(((got[:, :32].square() + got[:, 32:].square() - 1).abs() <= 2.0 ** -9).all())
    if f < 2e9:
        for i, p in enumerate(pos.tolist()):
            c, s = turned(L(1), L(0), p, freqs.cpu().numpy())
            want = torch.tensor([float(x) for x in (*c, *s)], dtype=torch.float64, device="cuda")
            assert bool(((got[i] - want).abs() <= 2.0 ** -12 + 2.0 ** -20).all()), (p, float((got[i] - want).abs().max()))


def test_codes_of_amplitudes_and_eps_next_to_a_border(P):
    """An amplitude and an eps that fp32 does not hold decide codes."""
    rng, n = np.random.default_rng(62), 32
    for _ in range(8):
        (_, x) = bf16(rng, 20, 200, 1)
        for side in (1, -1):
            amp = float(L(border(x[0] * 1.1)) / L(x[0]) * (1 + side * L(2) ** -30))
            row = np.full(2 * n, x[0])
            row[0] = 256.0                                         # the scale is 1
            got = one_token(P, torch.from_numpy(row).to(torch.bfloat16)[None], np.zeros(n), amplitude=amp)[0]
            assert np.array_equal(got[0, 1:n], nearest(L(x[0]) * L(amp) * np.ones(n - 1, dtype=L)))
            # x w / sqrt(x^2 / hd + eps)
            w = np.float32(rng.uniform(30, 60))
            y = border(float(w) / math.sqrt(1 / 64 + 0.1 * rng.uniform(0.5, 2)))
            eps = float((L(w) / (L(y) * (1 + side * L(2) ** -31))) ** 2 - L(1) / 64)
            one = torch.zeros(1, 64, dtype=torch.bfloat16)
            one[0, 5] = 1.0
            wk = torch.full((64,), float(w), device="cuda")
            got, _, ks, _ = one_token(P, one, None, eps=eps, k_norm=wk)
            want = nearest(L(w) / np.sqrt(L(1) / 64 + L(eps)) / ks[0])
            assert got[0, 5] == want and not np.delete(got[0], 5).any()


def test_scales_next_to_a_border(P):
    """Blocks whose largest value is 448 times a power of two, 2^-31 of it more or less: the scale goes by the exact value."""
    rng, KH, n = np.random.default_rng(63), 16, 32
    for _ in range(12):
        rows, f, top = np.zeros((KH, 2 * n)), np.zeros(n), np.zeros(KH, dtype=L)
        for h in range(KH):
            while True:
                (_, x), (_, y) = bf16(rng, 300, 640, 1), bf16(rng, -400, 400, 1)
                phi = np.arctan2(L(y[0]), L(x[0]))
                r = np.sqrt(L(x[0]) ** 2 + L(y[0]) ** 2)
                if 448 / math.cos(0.3) < r < 448 / math.cos(0.7):
                    break
            t = np.arccos(448 * (1 + L(2) ** -31 * (1 if h % 2 else -1)) / r) - phi
            f[h] = np.float64(t)
            rows[h, h], rows[h, n + h] = x[0], y[0]
            top[h] = np.abs(turned(L(x[0]), L(y[0]), 1, f[h:h + 1])).max()
        assert bool((np.abs(top / 448 - 1) > L(2) ** -33).all())
        got, _, ks, vs = one_token(P, torch.from_numpy(rows).to(torch.bfloat16), f, position=1)
        assert np.array_equal(ks, np.where(top > 448, 2, 1).astype(L)), (ks, top - 448)
        want = np.where(top > 448, 224, 448)
        assert np.array_equal(np.abs(got).max(1), want.astype(L))


def test_codes_under_an_earlier_scale_of_any_kind(P):
    """Earlier tokens' scales that are no powers of two: they stay if they are larger, and the new codes are the nearest under them."""
    rng, KH, hd = np.random.default_rng(64), 32, 64
    for _ in range(6):
        rows = np.zeros((KH, hd))
        scale = np.zeros(KH, dtype=np.float32)
        for h in range(KH):
            x = torch.from_numpy(rng.uniform(0.5, 1, hd)).to(torch.bfloat16).double().numpy()
            near = np.float32(x[0] / border(rng.uniform(60, 105)))   # the largest value is below 224 scales, so this scale stays
            while True:   # a scale that takes the first value next to a border, and none to a tie
                near = np.nextafter(near, np.float32(2))
                y = x.astype(L) / L(near)
                step = L(2) ** (np.floor(np.log2(y)) - 3)
                if bool((np.abs(y / step % 1 - 0.5) > L(2) ** -40).all()):
                    break
            rows[h], scale[h] = x, near
        before = torch.from_numpy(scale).cuda()
        k, v, ks, vs = one_token(P, torch.from_numpy(rows).to(torch.bfloat16), None, ctx=3, before=before)
        assert np.array_equal(ks, scale.astype(L)) and np.array_equal(vs, scale.astype(L))
        want = nearest(rows.astype(L) / scale.astype(L)[:, None])
        assert np.array_equal(k, want) and np.array_equal(v, want), (int((k != want).sum()), int((v != want).sum()))
    # and where they grow, the earlier codes are the nearest to what they were
    codes = torch.arange(127, device="cuda").to(torch.uint8)[:112].view(1, 1, 1, 112).expand(1, KH, 16, 112).contiguous()
    k_pages, v_pages = codes.view(E4M3).clone(), codes.view(E4M3).clone()
    old = np.zeros(KH, dtype=np.float32)
    for h in range(KH):   # code 36 (3.0 = 1.5 x 2) or so times old is next to a border under the scale 1
        c = E4M3_VALUES[rng.integers(60, 100)]
        y = border(float(c) * rng.uniform(16.5 / float(c), 0.99)) if c > 17 else None
        old[h] = np.nextafter(np.float32(0.7 if y is None else y / float(c)), np.float32(2))
    ks, vs = (torch.from_numpy(old).cuda().view(1, KH, 1).clone() for _ in range(2))
    x = torch.full((1, KH, 112), 300.0, dtype=torch.bfloat16, device="cuda")
    P.cache_append(x, x, k_pages, v_pages, ints(0).view(1, 1), ints(16), k_scales=ks, v_scales=vs)
    assert bool((ks == 1).all())
    y = E4M3_VALUES[:112][None] * old.astype(L)[:, None]
    d = np.abs(y[..., None] - E4M3_VALUES)
    want = E4M3_VALUES[d.argmin(-1)]
    two = np.partition(d, 1, axis=-1)
    clear = two[..., 1] - two[..., 0] > np.abs(y) * L(2) ** -44     # ties aside
    for pages in (k_pages, v_pages):
        got = pages[0, :, 0].float().cpu().numpy().astype(L)
        assert np.array_equal(got[clear], want[clear])


@pytest.mark.parametrize("hd,n,interleaved", [(128, 16, False), (64, 8, True), (64, 0, False), (96, 5, False)])
def test_codes_of_infinities_under_a_norm(P, hd, n, interleaved):
    """A key with an infinity is NaN where that reaches and zero elsewhere, whatever the tokens beside it hold; one call and one by one."""
    g, T, KH = gen(65), 1024, 4
    pool = Pool(g, torch.bfloat16, True, KH, hd, 64, [T])
    one = pool.clone()
    k, v = (rand(g, T, KH, hd, dtype=torch.bfloat16, scale=2.0) for _ in range(2))
    at = torch.arange(T, device="cuda") % 16 == 5
    k[at, :, 3] = math.inf
    k[at, 1, hd - 1] = -math.inf
    f = P.rotary_frequencies(2 * n, 1e4, device="cuda")[0] if n else None
    kw = {"freqs": f, "interleaved": interleaved, "k_norm": 1 + 0.3 * torch.randn(hd, generator=g, device="cuda")}
    P.cache_append(k, v, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, **kw)
    p = torch.arange(T, device="cuda")
    codes = pool.k.transpose(1, 2)[pool.tables[0].long()[p // 64], p % 64].float()       # [T, KH, hd]
    want = torch.zeros(KH, hd, dtype=torch.bool, device="cuda")
    want[:, 3] = True
    want[1, hd - 1] = True
    if n > 3:
        want[:, 3 + n if not interleaved else 2] = True
    assert torch.equal(torch.isnan(codes[at]), want.expand(int(at.sum()), KH, hd))
    assert not bool(codes[at].nan_to_num(0.0).any()) and bool(torch.isfinite(codes[~at]).all())
    for t in range(0, T):
        P.cache_append(k[t:t + 1], v[t:t + 1], one.k, one.v, one.tables, ints(t + 1), **one.kw, **kw)
    # the scale of a block that grows token by token ends as that of the whole block; the last token's codes were written under it
    assert torch.equal(one.ks, pool.ks)
    last = torch.arange(15, T, 16, device="cuda")
    rows = lambda x: bits(x.transpose(1, 2)[pool.tables[0].long()[last // 64], last % 64])  # noqa: E731
    assert torch.equal(rows(one.k), rows(pool.k))


def test_codes_beyond_fp32(P):
    """Turned values that fp32 does not hold are NaN and do not count for the scale, heads whose sum of squares it does not hold are
    normed to zero, whatever the tokens beside them hold."""
    g, T, KH, hd, top = gen(67), 1024, 4, 64, torch.finfo(torch.float32).max
    pool = Pool(g, torch.bfloat16, True, KH, hd, 64, [T])
    k = (torch.randn(T, KH, hd, generator=g, device="cuda") * 1.2e38).clamp(-3.3e38, 3.3e38).to(torch.bfloat16)
    f, p = P.rotary_frequencies(hd, 1e4, device="cuda")[0], torch.arange(T, device="cuda")
    P.cache_append(k, k, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, freqs=f)
    t, (a, b) = (p.double()[:, None] * f)[:, None], k.double().split(hd // 2, -1)
    y = torch.cat([a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()], -1)
    page, row = pool.tables[0].long()[p // 64], p % 64
    codes, scale = pool.k.transpose(1, 2)[page, row].double(), pool.ks[page, :, row // 16].double()
    # sine, cosine, product and sum: off by (|a| + |b|) 3 2^-24 <= 2 (3.3e38) 3 2^-24 < 2^-21 of fp32's largest
    over, fits = y.abs() > top * (1 + 2.0 ** -21), y.abs() < top * (1 - 2.0 ** -21)
    assert int(over.sum()) > 20 and bool((over | fits).all()) and torch.equal(torch.isnan(codes), over)
    need = torch.exp2(torch.ceil(torch.log2(torch.where(fits, y.abs(), 0.0).view(T // 16, 16, KH, hd).amax((1, 3)) / 448)))
    assert torch.equal(scale, need.repeat_interleave(16, 0))
    step = torch.exp2(torch.clamp(torch.floor(torch.log2((y / scale[..., None]).abs().clamp(min=2.0 ** -30))), min=-6) - 3)
    u = y / scale[..., None] / step
    clear = fits & (((u - u.floor()) - 0.5).abs() > 2.0 ** -33 * torch.hypot(a, b).repeat(1, 1, 2) / scale[..., None] / step)
    # (token 0 is not turned, and of bf16's values, of 8 bits, one in 16 lies between two codes)
    assert torch.equal(codes[clear], (torch.round(u) * step)[clear]) and int((fits & ~clear)[1:].sum()) < 8
    # heads of 2^70 beside ordinary ones
    k = rand(g, T, KH, hd, dtype=torch.bfloat16)
    large = p % 16 == 9
    k[large] = (k[large].float() * 2.0 ** 70).to(torch.bfloat16)
    P.cache_append(k, k, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, freqs=f, k_norm=torch.ones(hd, device="cuda"))
    codes = pool.k.transpose(1, 2)[page, row].double()
    assert not bool(codes[large].any()) and bool(torch.isfinite(codes).all()) and bool((codes[~large].abs().amax(-1) > 0).all())


@pytest.mark.parametrize("ctx", [0, 5, 15])
def test_codes_are_the_64_bit_values_rounded(P, ctx):
    """Half a million codes under an amplitude and an eps that fp32 does not hold, at far positions and in blocks begun before: those
    that 64 bits give, but for values within 2^-33 of their pair of a border."""
    g, T, KH, hd, amp, eps = gen(66), 1024, 4, 128, 1.1, 1.1e-5
    pool = Pool(g, torch.bfloat16, True, KH, hd, 64, [T + ctx])
    k = rand(g, T, KH, hd, dtype=torch.bfloat16, scale=2.0)
    f = P.rotary_frequencies(hd, 1e6, device="cuda")[0]
    w = 1 + 0.3 * torch.randn(hd, generator=g, device="cuda")
    pos = torch.randint(0, 1 << 17, (T,), generator=g, device="cuda").int()
    old = pool.ks[int(pool.tables[0, 0]), :, 0].double()
    P.cache_append(k, k, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, freqs=f, k_norm=w, amplitude=amp, eps=eps, positions=pos)
    x = k.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    t = (pos.double()[:, None] * f)[:, None]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    y = amp * torch.cat([a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()], -1)
    p = torch.arange(ctx, T + ctx, device="cuda")
    page, row = pool.tables[0].long()[p // 64], p % 64
    scale = pool.ks[page, :, row // 16].double()
    for blk in range(p[0] // 16, p[-1] // 16 + 1):
        m = p // 16 == blk
        need = torch.exp2(torch.ceil(torch.log2(y[m].abs().amax((0, 2)) / 448)))
        assert torch.equal(scale[m][0], torch.maximum(need, old) if ctx and blk == 0 else need)
    y = y / scale[..., None]
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))), min=-6) - 3)
    u, pair = y / step, amp * torch.hypot(a, b).repeat(1, 1, 2) / scale[..., None] / step
    clear = ((u - u.floor()) - 0.5).abs() > 2.0 ** -33 * pair        # t is off by 2^17 2^-53 radians at most here
    got = pool.k.transpose(1, 2)[page, row].double()
    want = torch.round(u) * step
    assert torch.equal(got[clear], want[clear]) and int((~clear).sum()) < 8


# ---- how they are called

def stride_words(*tensors):
    return (ctypes.c_int64 * 32)(*[s for t, n in tensors for s in t.stride()[:n]])


def test_entries_by_their_argument_lists(P, gpu):
    """The four C entries, every argument of a type another one: the bits of the Python calls."""
    g, H, KH, hd, page, T, B, n = gen(71), 6, 2, 64, 32, 9, 3, 2
    f = P.rotary_frequencies(48, 1e4, device="cuda")[0]
    wq, wk, sinks = (1 + 0.3 * torch.randn(m, generator=g, device="cuda") for m in (hd, hd, H))
    y = rand(g, T, H + 2 * KH, hd, dtype=torch.float16, scale=2.0)
    q, k, v = y[:, :H], y[:, H:H + KH], y[:, H + KH:]
    pos, stream = torch.randint(0, 9999, (T,), generator=g, device="cuda").int(), torch.cuda.current_stream().cuda_stream
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    amp, eps = 1.25, 0.5 ** 10                                      # of fp32
    # rotation
    want = P.rotary(q, k, pos, f, interleaved=True, amplitude=amp, q_norm=wq, k_norm=wk, eps=eps)
    got = torch.full_like(y, 9.0)[:, :H], torch.full((KH, T, hd), 9.0, dtype=torch.float16, device="cuda").transpose(0, 1)
    st = stride_words((q, 2), (k, 2), (got[0], 2), (got[1], 2))
    assert gpu.tg_rotary(1, at(q), at(k), at(got[0]), at(got[1]), at(pos), at(f), at(wq), at(wk), T, H, KH, hd, len(f), 1, amp, eps, st, stream) == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for codes in (True, False):
        a = Pool(g, torch.float16, codes, KH, hd, page, [100, 70, 41])
        if codes:
            a.vs = a.vs.permute(2, 0, 1).contiguous().permute(1, 2, 0)
        a.v = a.v.view(torch.uint8 if codes else torch.int16).transpose(1, 2).contiguous().transpose(1, 2).view(a.v.dtype)
        wide = torch.full((B, a.tables.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
        wide[:, :a.tables.shape[1]] = a.tables
        a.tables = wide[:, :a.tables.shape[1]]
        b, cu = a.clone(), ints(0, 4, 5, 9)
        b.v = b.v.view(torch.uint8 if codes else torch.int16).transpose(1, 2).contiguous().transpose(1, 2).view(b.v.dtype)
        b.tables = wide[:, :a.tables.shape[1]]
        none = torch.empty_strided((1, 1, 1), (1, 1, 1))
        cache = lambda p: ((p.k, 3), (p.v, 3), (none if p.ks is None else p.ks, 3), (none if p.vs is None else p.vs, 3), (p.tables, 1))  # noqa: E731
        pb, cols = 8 if codes else 16, a.tables.shape[1]
        # appending
        want = P.cache_append(k, v, a.k, a.v, a.tables, a.lens, cu, **a.kw, freqs=f, positions=pos, amplitude=amp, q=q, q_norm=wq, k_norm=wk,
                              eps=eps)
        out = torch.full_like(y, 9.0)[:, :H]
        st = stride_words((q, 2), (k, 2), (v, 2), (out, 2), *cache(b))
        assert gpu.tg_paged_append(1, pb, at(q), at(k), at(v), at(out), at(b.k), at(b.v), at(b.ks), at(b.vs), at(b.tables), at(b.lens), at(cu), at(pos),
                                   at(f), at(wq), at(wk), T, B, b.n, page, cols, H, KH, hd, len(f), 0, amp, eps, st, stream) == 0
        assert torch.equal(out, want) and torch.equal(bits(a.k), bits(b.k)) and torch.equal(bits(a.v), bits(b.v))
        assert not codes or (torch.equal(a.ks, b.ks) and torch.equal(a.vs, b.vs))
        # attention, whole and cut
        x = rand(g, B, n, H, hd, dtype=torch.float16)
        for max_len, window in ((128, 30), (128, 0), (99, 0)):
            want = P.attention_paged(x, a.k, a.v, a.tables, a.lens, **a.kw, max_len=max_len, window=window, sinks=sinks, scale=0.25)
            out = torch.full((H, B, n, hd), 9.0, dtype=torch.float16, device="cuda").permute(1, 2, 0, 3)
            size = gpu.tg_attention_paged_workspace(pb, B, n, max_len, window, H, KH, hd)
            ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
            st = stride_words((x, 3), (out, 3), *cache(b))
            assert gpu.tg_attention_paged(1, pb, at(x), at(b.k), at(b.v), at(b.ks), at(b.vs), at(out), at(b.tables), at(b.lens), at(sinks), B, n, b.n, page,
                                          cols, max_len, H, KH, hd, st, window, 0.25, at(ws), size, stream) == 0
            assert torch.equal(out, want)
        # a unit's tiles in several pieces
        long = Pool(g, torch.float16, codes, KH, hd, page, [2000, 70, 1500])
        want = P.attention_paged(x, long.k, long.v, long.tables, long.lens, **long.kw, sinks=sinks, scale=0.25, max_len=2000)
        size = gpu.tg_attention_paged_workspace(pb, B, n, 2000, 0, H, KH, hd)
        assert size > 0
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        st = stride_words((x, 3), (out, 3), *cache(long))
        assert gpu.tg_attention_paged(1, pb, at(x), at(long.k), at(long.v), at(long.ks), at(long.vs), at(out), at(long.tables), at(long.lens), at(sinks), B, n,
                                      long.n, page, long.tables.shape[1], 2000, H, KH, hd, st, 0, 0.25, at(ws), size, stream) == 0
        assert torch.equal(out, want)
        # reading back
        cu = ints(0, 40, 70, 111)
        want = P.cache_gather(a.k, a.v, a.tables, cu, 111, **a.kw, dtype=torch.float16)
        ko, vo = torch.full((111, KH, hd), 9.0, dtype=torch.float16, device="cuda"), torch.full((KH, 111, hd), 9.0, dtype=torch.float16, device="cuda").transpose(0, 1)
        st = stride_words((ko, 2), (vo, 2), *cache(b))
        assert gpu.tg_paged_gather(1, pb, at(b.k), at(b.v), at(b.ks), at(b.vs), at(b.tables), at(cu), at(ko), at(vo), 111, B, b.n, page, cols, KH, hd, st,
                                   stream) == 0
        assert torch.equal(ko, want[0]) and torch.equal(vo, want[1])
    assert tg.last_error(gpu)[0] in (0, 3)


def refusal_tensors():
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    return {"q": z(4, 4, 64), "k": z(4, 2, 64), "f": z(32, dt=torch.float64), "i": ints(1, 2, 3, 4), "pages": z(3, 2, 32, 64),
            "codes": z(3, 2, 32, 64, dt=E4M3), "scales": z(3, 2, 2, dt=torch.float32) + 1, "tables": z(4, 2, dt=torch.int32)}


def test_broadcast_scales_and_tables_are_refused(P):
    t = refusal_tensors()
    q, k, i, codes, scales, tables = (t[n] for n in ("q", "k", "i", "codes", "scales", "tables"))
    for s in (scales[:1].expand(3, 2, 2), scales[:, :1].expand(3, 2, 2), scales[..., :1].expand(3, 2, 2)):
        for kw in ({"k_scales": s, "v_scales": scales}, {"k_scales": scales, "v_scales": s}):
            for call in (lambda: P.attention_paged(q, codes, codes, tables, i, **kw), lambda: P.cache_append(k, k, codes, codes, tables, i, **kw),
                         lambda: P.cache_gather(codes, codes, tables, ints(0, 1, 2, 3, 4), 4, **kw)):
                with pytest.raises(ValueError, match="strides of scales"):
                    call()
    kw, one = {"k_scales": scales, "v_scales": scales}, tables[:1].expand(4, 2)
    for call in (lambda: P.attention_paged(q, codes, codes, one, i, **kw), lambda: P.cache_append(k, k, codes, codes, one, i, **kw),
                 lambda: P.cache_gather(codes, codes, one, ints(0, 1, 2, 3, 4), 4, **kw)):
        with pytest.raises(ValueError, match="stride of tables"):
            call()


def test_numbers_that_are_none_are_refused(P):
    """max_len, window, scale, total, eps and amplitude of other kinds: ValueError, and numpy's whole numbers count as such."""
    t = refusal_tensors()
    q, k, f, i, pages, tables = (t[n] for n in ("q", "k", "f", "i", "pages", "tables"))
    for kw in ({"max_len": 2.5}, {"max_len": "9"}, {"max_len": math.nan}, {"max_len": [3]}, {"window": 1.5}, {"window": "2"}, {"window": None},
               {"scale": "1"}, {"scale": [1.0]}, {"scale": math.inf}):
        with pytest.raises(ValueError):
            P.attention_paged(q, pages, pages, tables, i, **kw)
    for kw in ({"eps": "x"}, {"eps": None}, {"amplitude": [1.0]}, {"interleaved": "yes"}):
        with pytest.raises(ValueError):
            P.rotary(q, k, i, f, **kw)
        with pytest.raises(ValueError):
            P.cache_append(k, k, pages, pages, tables, i, freqs=f, **kw)
    for total in (4.0, "4", None, -1):
        with pytest.raises(ValueError):
            P.cache_gather(pages, pages, tables, ints(0, 1, 2, 3, 4), total)
    want = P.attention_paged(q, pages, pages, tables, i, max_len=40, window=3)
    assert torch.equal(P.attention_paged(q, pages, pages, tables, i, max_len=np.int64(40), window=np.int32(3)), want)
    assert P.cache_gather(pages, pages, tables, ints(0, 1, 2, 3, 4), np.int64(4))[0].shape == (4, 2, 64)


def test_dual_tensors_are_refused(P):
    """Forward-mode derivatives would be lost without a word: refused, here and by the attention operators beside."""
    from torch.autograd import forward_ad as fw

    from tinygiant_b200 import attention as A
    t = refusal_tensors()
    q, k, f, i, pages, tables = (t[n] for n in ("q", "k", "f", "i", "pages", "tables"))
    cache, lens = torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16, device="cuda"), ints(1, 2, 3, 4)
    w = torch.zeros(4, 2, 8, device="cuda")
    calls = [(q, lambda d: P.rotary(d, k, i, f)), (k, lambda d: P.rotary(q, d, i, f)), (f, lambda d: P.rotary(q, k, i, d)),
             (q, lambda d: P.rotary(q, k, i, f, out=(d, k))),
             (k, lambda d: P.cache_append(d, k, pages, pages, tables, i)), (k, lambda d: P.cache_append(k, d, pages, pages, tables, i)),
             (pages, lambda d: P.cache_append(k, k, d, pages, tables, i)), (q, lambda d: P.cache_append(k, k, pages, pages, tables, i, q=d)),
             (q, lambda d: P.attention_paged(d, pages, pages, tables, i)), (pages, lambda d: P.attention_paged(q, pages, d, tables, i)),
             (pages, lambda d: P.cache_gather(pages, d, tables, ints(0, 1, 2, 3, 4), 4)),
             (q, lambda d: A.attention_prompt(d, k, k, ints(0, 4))), (k, lambda d: A.attention_prompt(q, k, d, ints(0, 4))),
             (q, lambda d: A.attention_shared(d, None, None, cache, cache, lens)), (cache, lambda d: A.attention_shared(q, None, None, cache, d, lens)),
             (cache, lambda d: A.cache_evict(cache, d, w, lens, 4, 1))]
    for x, call in calls:
        call(x.clone())
        with fw.dual_level():
            call(x.clone())                                        # no tangent, no refusal
            with pytest.raises(ValueError, match="no backward pass"):
                call(fw.make_dual(x.clone(), torch.ones_like(x)))


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_two_calls_at_once(P, codes):
    """Two streams append to and attend over one pool, each for its own sequences, under inference mode: the bits of one after the other."""
    g, H, KH, hd, n = gen(72), 16, 2, 128, 6
    lens = [1500, 700, 33, 2100, 16, 900]
    pool = Pool(g, torch.bfloat16, codes, KH, hd, 16, lens)
    q, k, v = (rand(g, n, h, hd, dtype=torch.bfloat16) for h in (H, KH, KH))
    f = P.rotary_frequencies(hd, device="cuda")[0]

    def half(p, rows):
        outs = []
        for _ in range(20):
            y = P.cache_append(k[rows], v[rows], p.k, p.v, p.tables[rows], p.lens[rows], **p.kw, freqs=f, q=q[rows])
            outs.append(P.attention_paged(y, p.k, p.v, p.tables[rows], p.lens[rows], **p.kw))
        return outs

    with torch.inference_mode():
        one, both = pool.clone(), pool.clone()
        want = half(one, slice(0, 3)) + half(one, slice(3, 6))
        streams, got = [torch.cuda.Stream() for _ in range(2)], []
        for s, rows in zip(streams, (slice(0, 3), slice(3, 6))):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got += half(both, rows)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(bits(one.k), bits(both.k)) and torch.equal(bits(one.v), bits(both.v))
