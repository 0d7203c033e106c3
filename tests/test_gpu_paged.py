"""The paged cache (tinygiant_b200.paged) against the definitions in 64 bits:
rotation, appending in 16 and 8 bits, attention over pages, reading them back,
a run of them together, and what they refuse.

Tolerances, element by element.  u is half a step of the type (2^-8 bf16,
2^-11 fp16, 2^-4 e4m3).
  Rotation: a row's norm and its weights are hd fp32 additions and a few more
  roundings, (hd + 16) 2^-24 of each value together; sine and cosine are off by 4
  2^-24 at most and the products and their sum by 3 2^-24; so with a pair (a, b)
  times the amplitude, (|a| + |b|) (hd + 24) 2^-24 (call it d), and the output's
  rounding u |y| (half of fp16's least step, 2^-25, below its normal values).
  Codes: |code scale - y| <= u |y|, or half of e4m3's least step, 2^-10 scale,
  and d (1 + u).  Scales, and codes rounded again, are exact.
  Attention: as test_gpu_attn_ops has it, |o - o64| <= u |o64| + (w + 2 delta)
  1.05 A, where the weights are rounded to fp16 (w = 2^-11) with pages of 8
  bits and to the type (w = u) else; delta = (hd + 16) 2^-23 S + 2^-18 has the
  base-2 logarithm of the values' scale (|log2| <= 32: 32 2^-23 ln 2 < 2^-18)
  that is added to each exponent."""
import ctypes
import math

import numpy as np
import pytest

import tinygiant_b200 as tg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def P(gpu):
    from tinygiant_b200 import paged
    return paged


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def ints(*x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def ends(lens):
    return ints(0, *np.cumsum(lens))


def bits(t):
    return t.contiguous().view(torch.uint8)


# ---- rotation

def rotate64(x, positions, freqs, interleaved, amplitude, norm, eps=1e-6):
    """Rotated rows and d, in 64 bits."""
    x, hd, n = x.double(), x.shape[-1], 0 if freqs is None else len(freqs)
    y = x if norm is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    out, d = y.clone(), torch.zeros_like(y) if norm is None else y.abs() * (hd + 16) * 2.0 ** -24
    if n:
        t = (positions.double()[:, None] * freqs)[:, None]
        lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
        a, b = y[..., lo], y[..., hi]
        out[..., lo], out[..., hi] = amplitude * (a * t.cos() - b * t.sin()), amplitude * (b * t.cos() + a * t.sin())
        d[..., lo] = d[..., hi] = (a.abs() + b.abs()) * abs(amplitude) * (hd + 24) * 2.0 ** -24
    return out, d


def near(got, want, d):
    u = U[got.dtype]
    tol = u * want.abs() + d + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    worst = ((got.double() - want).abs() - tol).max() if got.numel() else torch.tensor(0.0)
    assert bool(((got.double() - want).abs() <= tol).all()), float(worst)


ROTARY = [     # tokens, heads, kv heads, head_dim, pairs, interleaved, norms
    (1, 1, 1, 8, 4, False, False), (3, 32, 4, 128, 64, False, True), (5, 64, 8, 64, 32, False, False), (2, 5, 0, 64, 8, True, True),
    (7, 28, 4, 128, 32, True, False), (4, 16, 16, 80, 10, False, True), (4, 16, 1, 80, 5, True, False), (6, 3, 2, 96, 48, False, True),
    (9, 100, 3, 72, 36, True, True), (300, 24, 8, 96, 12, False, False), (2, 8, 2, 40, 0, False, True), (3, 8, 2, 128, 1, False, False),
    (3, 7, 5, 16, 7, False, True), (1000, 8, 2, 64, 16, False, False), (2, 130, 70, 64, 31, False, True)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "-".join(map(str, c)))
def test_rotary_matches_definition(P, case, dtype):
    T, H, KH, hd, n, inter, norms = case
    g, dt = gen(1), DT[dtype]
    q, k = rand(g, T, H, hd, dtype=dt, scale=2.0), rand(g, T, KH, hd, dtype=dt) if KH else None
    f, amp = P.rotary_frequencies(2 * n, 1e6, device="cuda")[0] if n else torch.zeros(0, dtype=torch.float64, device="cuda"), 1.25
    pos = torch.randint(0, 200000, (T,), generator=g, device="cuda").int()
    w = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") if norms else None for _ in range(2)]
    qo, ko = P.rotary(q, k, pos, f, interleaved=inter, amplitude=amp, q_norm=w[0], k_norm=w[1])
    near(qo, *rotate64(q, pos, f, inter, amp, w[0]))
    assert qo.is_contiguous() and (ko is None) == (k is None)
    if k is not None:
        near(ko, *rotate64(k, pos, f, inter, amp, w[1]))
    if not norms:
        assert torch.equal(qo[..., 2 * n:], q[..., 2 * n:])
    # in place, and one norm alone
    qi = q.clone()
    ki = None if k is None else k.clone()
    assert P.rotary(qi, ki, pos, f, interleaved=inter, amplitude=amp, q_norm=w[0], k_norm=w[1], out=(qi, ki))[0] is qi
    assert torch.equal(qi, qo) and (k is None or torch.equal(ki, ko))
    if norms and k is not None:
        q1, k1 = P.rotary(q, k, pos, f, interleaved=inter, amplitude=amp, k_norm=w[1])
        near(q1, *rotate64(q, pos, f, inter, amp, None))
        assert torch.equal(k1, ko)


def test_rotary_of_far_positions_and_signs(P):
    """Angles of positions up to 2^31 and below zero; frequencies of fp64 that fp32 does not hold."""
    g = gen(2)
    pos = ints(0, 1, -1, 16777217, 2147483647, -2147483647, 123456789, 99999999)
    q = rand(g, len(pos), 4, 64, dtype=torch.float16)
    f = torch.rand(32, generator=g, device="cuda", dtype=torch.float64)
    for inter in (False, True):
        got, _ = P.rotary(q, None, pos, f, interleaved=inter)
        # p f in turns is off by 2^-53 of up to 2^28.4 turns, twice: 2^-21 radians; here p f in radians is off by 2^-22
        want, d = rotate64(q, pos, f, inter, 1.0, None)
        near(got, want, d * (1 + 12 / 88))
    zero, _ = P.rotary(q, None, torch.zeros_like(pos), f)
    assert torch.equal(zero, q)


def test_rotary_keeps_what_is_not_finite_where_it_is(P):
    g = gen(3)
    q = rand(g, 4, 2, 96, dtype=torch.bfloat16)
    q[1, 0, 3], q[2, 1, 40], q[3, 0, 90], q[3, 1, 91] = math.nan, math.inf, math.inf, math.nan
    f = P.rotary_frequencies(64, device="cuda")[0]
    got, _ = P.rotary(q, None, ints(5, 6, 7, 8), f)
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[1, 0, [3, 35]] = want[2, 1, [40, 8]] = want[3, 0, 90] = want[3, 1, 91] = True
    assert torch.equal(bad, want) and got[3, 0, 90] == math.inf


def test_rotary_strided_views(P):
    g, f = gen(4), None
    y = rand(g, 37, 12, 64, dtype=torch.float16)
    f, pos = P.rotary_frequencies(64, device="cuda")[0], torch.arange(37, device="cuda").int()
    want = P.rotary(y[:, :8].contiguous(), y[:, 8:10].contiguous(), pos, f)
    back = torch.full_like(y, 9.0)
    P.rotary(y[:, :8], y[:, 8:10], pos, f, out=(back[:, 2:10], back[:, 10:]))
    assert torch.equal(back[:, 2:10], want[0]) and torch.equal(back[:, 10:], want[1]) and bool((back[:, :2] == 9).all())
    t = y[:, :8].transpose(0, 1).contiguous().transpose(0, 1)                   # head-major
    assert torch.equal(P.rotary(t, None, pos, f)[0], want[0])
    v = y._version
    P.rotary(y[:, :8], None, pos, f, out=(y[:, :8], None))
    assert y._version > v


# ---- pools

class Pool:
    """Pages of random contents, tables of random pages, lengths."""

    def __init__(self, g, dt, codes, KH, hd, page, lens, spare=2, cols=0, spread=0.0):
        need = [-(-n // page) for n in lens]
        self.n, self.page, self.dt, self.codes = sum(need) + spare, page, dt, codes
        order = torch.randperm(self.n, generator=g, device="cuda").int()
        self.tables = torch.full((len(lens), max([*need, cols, 1])), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, m in enumerate(need):
            self.tables[b, :m] = order[at:at + m]
            at += m
        self.lens = ints(*lens)
        if codes:
            def one(scale):
                y = torch.randn(self.n, KH, page, hd, generator=g, device="cuda") * scale
                s = torch.exp2(torch.randint(-6, -3, (self.n, KH, page // 16), generator=g, device="cuda").float())
                s *= torch.exp2(torch.round(spread * torch.randn(s.shape, generator=g, device="cuda")).clamp(-20, 20))
                y = y * 2.0 ** 5 if spread else y / s.repeat_interleave(16, 2)[..., None]
                return y.clamp(-448, 448).to(E4M3), s
            (self.k, self.ks), (self.v, self.vs) = one(1.0), one(1.0)
            if spread:
                self.ks = torch.full_like(self.ks, 2.0 ** -5)
        else:
            self.k, self.v = rand(g, self.n, KH, page, hd, dtype=dt), rand(g, self.n, KH, page, hd, dtype=dt)
            self.ks = self.vs = None

    @property
    def kw(self):
        return {"k_scales": self.ks, "v_scales": self.vs}

    def values(self, x, b, n):
        """The first n positions of sequence b, [KH, n, hd] in 64 bits; zeros where there is no page."""
        pages, s = (self.k, self.ks) if x == "k" else (self.v, self.vs)
        y = pages.double() if s is None else pages.double() * s.double().repeat_interleave(16, 2)[..., None]
        j = torch.arange(n, device="cuda")
        t = self.tables[b].long()[j // self.page]
        ok = (t >= 0) & (t < self.n)
        return torch.where(ok[None, :, None], y[t.clamp(0, self.n - 1), :, j % self.page].transpose(0, 1), 0.0)

    def clone(self):
        c = object.__new__(Pool)
        c.__dict__ = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in self.__dict__.items()}
        return c


# ---- appending

def places(pool, b, first, n):
    """(page, row) of positions first .. first + n - 1, those that have one."""
    cols = pool.tables.shape[1]
    out = []
    for p in range(first, first + n):
        if 0 <= p < cols * pool.page:
            t = int(pool.tables[b, p // pool.page])
            if 0 <= t < pool.n:
                out.append((p, t, p % pool.page))
    return out


def check_append(before, after, k64, dk, v64, cu, new):
    """Pools before and after new[b] tokens of sequence b ended at lens[b]; k64, v64 [T, KH, hd] what they hold, off by dk and 0."""
    for x, want, d in (("k", k64, dk), ("v", v64, torch.zeros_like(v64))):
        pages, old = getattr(after, x), getattr(before, x)
        scales, old_scales = getattr(after, x + "s"), getattr(before, x + "s")
        same = torch.ones(old.shape[0], old.shape[2], dtype=torch.bool, device="cuda")       # rows that no token touches
        same_scale = None if scales is None else torch.ones(old.shape[0], old.shape[2] // 16, dtype=torch.bool, device="cuda")
        for b, n in enumerate(new):
            first = int(after.lens[b]) - n
            here = places(after, b, first, n)
            if not here:
                continue
            p, t, r = (torch.tensor(z, device="cuda") for z in zip(*here))
            rows = cu[b] + p - first
            same[t, r] = False
            if scales is None:
                near(pages[t, :, r], want[rows], d[rows])
                continue
            for blk in torch.unique(p // 16).tolist():
                m = p // 16 == blk
                page, row0, start = int(t[m][0]), blk * 16 % after.page, max(0, first - blk * 16)
                y, dy = want[rows[m]].transpose(0, 1), d[rows[m]].transpose(0, 1)            # [KH, tokens, hd]
                fine = torch.isfinite(y)
                amax = torch.where(fine, y.abs(), 0.0).amax((1, 2))
                need = torch.exp2(torch.ceil(torch.log2((amax / 448).clamp(min=2.0 ** -117))))
                edge = (amax / 448 / need - 0.5).abs().min(), (amax / 448 / need - 1).abs().min()
                assert min(map(float, edge)) > 1e-5 or float(dy.max()) == 0.0                # this test's data are off the border
                s_old = old_scales[page, :, row0 // 16].double()
                s = torch.maximum(need, s_old) if start else need
                assert torch.equal(scales[page, :, row0 // 16].double(), s), (x, b, blk)
                same_scale[page, row0 // 16] = False
                codes = pages[page, :, row0 + start:row0 + start + y.shape[1]].double()
                got, sh = codes * s[:, None, None], s[:, None, None]
                tol = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * sh) + dy * (1 + 2.0 ** -4)
                assert bool(((got - y).abs() <= tol)[fine].all()) and bool(torch.isnan(codes)[~fine].all())
                assert bool(torch.isfinite(codes)[fine].all())
                if start:
                    again = (old[page, :, row0:row0 + start].float() * (s_old / s).float()[:, None, None]).to(E4M3)
                    assert torch.equal(bits(pages[page, :, row0:row0 + start]), bits(again))
                    same[page, row0:row0 + start] = False
        assert torch.equal(bits(pages.transpose(1, 2)[same]), bits(old.transpose(1, 2)[same]))
        if scales is not None:
            assert torch.equal(scales.transpose(1, 2)[same_scale], old_scales.transpose(1, 2)[same_scale])


APPEND = [     # heads (0: no q), kv heads, head_dim, page, new tokens, tokens before, pairs, interleaved, norms
    (32, 4, 128, 16, [1, 1, 1], [0, 15, 16], 64, False, True),
    (8, 2, 64, 64, [1, 0, 1, 1], [63, 5, 64, 40], 32, False, False),
    (0, 1, 128, 32, [17, 1, 40, 0, 3], [3, 31, 0, 7, 30], 32, True, True),
    (4, 4, 96, 16, [16, 16, 32], [0, 8, 16], 12, False, False),
    (5, 5, 80, 256, [300, 2], [250, 14], 10, False, True),
    (64, 8, 64, 16, [4] * 9, [0, 1, 12, 13, 14, 15, 16, 17, 31], 32, False, False),
    (16, 1, 16, 128, [5, 130, 1], [11, 120, 0], 8, False, True),
    (28, 4, 128, 64, [200, 77], [0, 500], 0, False, False),
    (0, 20, 32, 16, [1] * 40, list(range(40)), 16, True, False),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c[:4])) + f"-{sum(c[4])}")
def test_append_matches_definition(P, case, codes, dtype):
    H, KH, hd, page, new, ctx, n, inter, norms = case
    g, dt = gen(11), DT[dtype]
    pool = Pool(g, dt, codes, KH, hd, page, [a + b for a, b in zip(new, ctx)])
    T = sum(new)
    y = rand(g, T, H + 2 * KH, hd, dtype=dt, scale=3.0)
    y *= torch.exp2(torch.randint(-3, 4, (T, 1, 1), generator=g, device="cuda")).to(dt)      # scales that have to grow, and not
    q, k, v = y.split([H, KH, KH], 1)
    f = P.rotary_frequencies(2 * n, device="cuda")[0] if n else None
    w = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") if norms else None for _ in range(2)]
    before = pool.clone()
    out = P.cache_append(k, v, pool.k, pool.v, pool.tables, pool.lens, ends(new), **pool.kw, freqs=f, interleaved=inter, amplitude=0.75,
                         q=q if H else None, q_norm=w[0], k_norm=w[1])
    pos = torch.cat([torch.arange(c, c + m, device="cuda") for m, c in zip(new, ctx)])
    cu = [0, *np.cumsum(new)]
    check_append(before, pool, *rotate64(k, pos, f, inter, 0.75, w[1]), v.double(), cu, new)
    if H:
        near(out, *rotate64(q, pos, f, inter, 0.75, w[0]))
    else:
        assert out is None
    # the same call again changes nothing: it is as if it had come once
    once = pool.clone()
    P.cache_append(k, v, pool.k, pool.v, pool.tables, pool.lens, ends(new), **pool.kw, freqs=f, interleaved=inter, amplitude=0.75,
                   k_norm=w[1])
    assert torch.equal(bits(pool.k), bits(once.k)) and torch.equal(bits(pool.v), bits(once.v))


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_append_of_tokens_without_a_place(P, codes):
    """Positions below zero and behind the table, pages outside the pool, rows of no sequence, more sequences than fit shared memory."""
    g, dt, KH, hd = gen(12), torch.bfloat16, 2, 64
    pool = Pool(g, dt, codes, KH, hd, 16, [40, 40, 40, 40], cols=4)
    pool.tables[1, 1], pool.tables[2, 0], pool.tables[2, 2] = -1, pool.n, 2147483647
    pool.lens = ints(3, 40, 40, 70)                                       # 10 new: from -7 on; .. ; .. ; up to 69 of 64 places
    new = [10, 30, 40, 10]
    before = pool.clone()
    T = sum(new) + 6                                                      # two rows before the first sequence, four behind the last
    q, k, v = (rand(g, T, h, hd, dtype=dt) for h in (4, KH, KH))
    cu = [2, *(2 + np.cumsum(new))]
    out = torch.full_like(q, 7.0)
    P.cache_append(k, v, pool.k, pool.v, pool.tables, pool.lens, ints(*cu), **pool.kw, q=q, out=out)
    check_append(before, pool, k.double(), torch.zeros_like(k, dtype=torch.float64), v.double(), cu, new)
    assert torch.equal(out[2:-4], q[2:-4]) and bool((out[:2] == 7).all()) and bool((out[-4:] == 7).all())
    # one token of each of many sequences, idle ones among them
    B = 1500
    lens = [int(x) for x in np.random.default_rng(0).integers(0, 3, B)]
    pool = Pool(g, dt, codes, KH, hd, 16, lens)
    before = pool.clone()
    k, v = (rand(g, B, KH, hd, dtype=dt) for _ in range(2))
    P.cache_append(k, v, pool.k, pool.v, pool.tables, pool.lens, **pool.kw)
    check_append(before, pool, k.double(), torch.zeros_like(k, dtype=torch.float64), v.double(), list(range(B + 1)), [1] * B)
    again = before.clone()
    P.cache_append(k, v, again.k, again.v, again.tables, again.lens, torch.arange(B + 1, device="cuda").int(), **again.kw)
    assert torch.equal(bits(again.k), bits(pool.k)) and torch.equal(bits(again.v), bits(pool.v))


def test_append_of_unusual_values(P):
    """Zeros, the least and largest numbers, infinities and NaN under 8-bit scales; a block whose earlier scale is far off."""
    g, KH, hd = gen(13), 2, 64
    pool = Pool(g, torch.bfloat16, True, KH, hd, 16, [16, 16, 16, 16, 16, 5])
    k, v = (rand(g, 81, KH, hd, dtype=torch.bfloat16) for _ in range(2))
    k[:16] = 0
    k[16:32] *= 2.0 ** -125
    k[32:48] *= 2.0 ** 120
    k[48:64, :, 5], v[48:64, :, 6] = math.nan, -math.inf
    k[64:80] = math.inf
    before = pool.clone()
    before.ks[int(pool.tables[5, 0]), :, 0] = pool.ks[int(pool.tables[5, 0]), :, 0] = 2.0 ** -30          # 4 codes shrink to nothing
    before.vs[int(pool.tables[5, 0]), :, 0] = pool.vs[int(pool.tables[5, 0]), :, 0] = 2.0 ** 30           # and this scale stays
    new = [16] * 5 + [1]
    P.cache_append(k, v, pool.k, pool.v, pool.tables, pool.lens, ends(new), **pool.kw)
    check_append(before, pool, k.double(), torch.zeros_like(k, dtype=torch.float64), v.double(), [0, *np.cumsum(new)], new)
    at = [int(t) for t in pool.tables[:, 0]]
    assert bool((pool.ks[at[0]] == 2.0 ** -117).all()) and not bool(pool.k[at[0]].float().any())
    assert bool((pool.ks[at[4]] == 2.0 ** -117).all()) and bool(torch.isnan(pool.k[at[4]].float()).all())
    assert bool((pool.vs[at[5], :, 0] == 2.0 ** 30).all())


def test_append_strided_views_and_positions(P):
    """Pools with tokens before heads, tables cut from wider ones, positions of their own, q in place."""
    g, KH, hd, page = gen(14), 3, 64, 32
    for codes in (True, False):
        a = Pool(g, torch.float16, codes, KH, hd, page, [50, 20, 33])
        b = a.clone()
        wide = torch.full((3, 7), -5, dtype=torch.int32, device="cuda")
        wide[:, 2:2 + a.tables.shape[1]] = a.tables
        b.k, b.v = (x.view(torch.uint8 if codes else torch.int16).transpose(1, 2).contiguous().transpose(1, 2).view(x.dtype) for x in (a.k, a.v))
        if codes:
            b.ks, b.vs = (x.permute(2, 1, 0).contiguous().permute(2, 1, 0) for x in (a.ks, a.vs))
        y = rand(g, 30, 6 + 2 * KH, hd, dtype=torch.float16)
        q, k, v = y[:, :6], y[:, 6:6 + KH], y[:, 6 + KH:]
        f, pos, cu = P.rotary_frequencies(64, device="cuda")[0], torch.randint(0, 9999, (30,), generator=g, device="cuda").int(), ints(0, 20, 21, 30)
        want = P.cache_append(k.contiguous(), v.contiguous(), a.k, a.v, a.tables, a.lens, cu, **a.kw, freqs=f, positions=pos, q=q.contiguous())
        assert torch.equal(want, P.rotary(q, None, pos, f)[0])
        got = P.cache_append(k, v, b.k, b.v, wide[:, 2:2 + a.tables.shape[1]], b.lens, cu, **b.kw, freqs=f, positions=pos, q=q, out=q)
        assert got is q and torch.equal(q, want)
        assert torch.equal(bits(a.k), bits(b.k)) and torch.equal(bits(a.v), bits(b.v))
        assert not codes or (torch.equal(a.ks, b.ks) and torch.equal(a.vs, b.vs))


# ---- reading back

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("KH,hd,page,lens", [(4, 128, 64, [100, 0, 1, 64, 65]), (8, 64, 16, [517, 1, 0, 300]), (1, 80, 32, [33]),
                                             (3, 96, 256, [700, 255]), (5, 16, 16, [1, 2, 3, 40])])
def test_gather_is_exact(P, KH, hd, page, lens, codes, dtype):
    g, dt = gen(21), DT[dtype]
    pool = Pool(g, dt, codes, KH, hd, page, lens)
    total = sum(lens)
    k, v = P.cache_gather(pool.k, pool.v, pool.tables, ends(lens), total, **pool.kw, dtype=dt)
    for x, got in (("k", k), ("v", v)):
        want = torch.cat([pool.values(x, b, n).transpose(0, 1) for b, n in enumerate(lens)]).to(dt)
        assert got.shape == (total, KH, hd) and torch.equal(got, want)
    # no place, no sequence, outputs of another shape in memory
    pool.tables[0, 0] = -1
    if len(lens) > 1:
        pool.tables[-1] = pool.n
    big = torch.full((2, KH, total + 5, hd), 3.0, dtype=dt, device="cuda").transpose(1, 2)
    cu = ends(lens) + 2
    P.cache_gather(pool.k, pool.v, pool.tables, cu, total + 5, **pool.kw, out=(big[0], big[1]))
    for i, x in enumerate("kv"):
        want = torch.cat([pool.values(x, b, n).transpose(0, 1) for b, n in enumerate(lens)]).to(dt)
        assert torch.equal(big[i, 2:2 + total], want) and bool((big[i, :2] == 3).all()) and bool((big[i, 2 + total:] == 3).all())


# ---- attention

def attend(q, k, v, ok, scale, sink):
    """q [n, hd], k, v [m, hd], ok [n, m]: outputs, the weighted mean of |v|, and delta, in 64 bits."""
    q = q.double()
    x = torch.where(ok, q @ k.T * scale, -math.inf)
    s = torch.where(ok, q.abs() @ k.abs().T * scale, 0.0)
    delta = (q.shape[1] + 16) * 2.0 ** -23 * (s.amax(1, keepdim=True) if s.shape[1] else s.new_zeros(len(q), 1)) + 2.0 ** -18
    if sink is not None:
        x = torch.cat([x, torch.full((len(q), 1), float(sink), dtype=torch.float64, device=q.device)], 1)
    p = torch.nan_to_num(torch.softmax(x, 1), nan=0.0)[:, :k.shape[0]]
    return p @ v, p @ v.abs(), delta


def paged_ref(pool, q, lens, window=0, sinks=None, scale=None):
    """Outputs, A and delta of q [B, n, H, hd]."""
    B, n, H, hd = q.shape
    KH = pool.k.shape[1]
    out, a, delta = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(3))
    for b, m in enumerate(lens):
        if m == 0:
            continue
        k, v = pool.values("k", b, m), pool.values("v", b, m)
        j = torch.arange(m, device=q.device)
        t = pool.tables[b].long()[j // pool.page]
        e = torch.arange(n, device=q.device)[:, None] + (m - n)
        ok = (j <= e) & (t >= 0) & (t < pool.n)
        if window:
            ok &= j > e - window
        for h in range(H):
            o = attend(q[b, :, h], k[h // (H // KH)], v[h // (H // KH)], ok, hd ** -0.5 if scale is None else scale,
                       None if sinks is None else sinks[h])
            out[b, :, h], a[b, :, h], delta[b, :, h] = o
    return out, a, delta


def check(got, want, a, delta, codes):
    u = U[got.dtype]
    tol = u * want.abs() + ((2.0 ** -11 if codes else u) + 2 * delta) * 1.05 * a + 2.0 ** -24
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


PAGED = [     # heads, kv heads, head_dim, page, queries, lens, window, sinks
    (1, 1, 64, 16, 1, [1], 0, False),
    (8, 2, 64, 16, 1, [0, 1, 2, 15, 16, 17, 31, 32, 33], 0, True),
    (32, 4, 128, 64, 1, [100, 33], 0, False),
    (32, 4, 128, 16, 1, [1000, 0, 257, 256, 255, 3000], 0, False),
    (64, 8, 64, 16, 4, [0, 3, 4, 5, 130, 1000, 517], 128, True),
    (16, 16, 96, 32, 1, [5, 700, 64], 0, True),
    (28, 4, 128, 128, 2, [300, 1, 2, 999], 0, False),
    (24, 8, 80, 256, 3, [600, 100], 50, False),
    (16, 1, 128, 16, 8, [777, 8, 20], 0, True),
    (128, 1, 64, 64, 2, [400, 65], 0, False),
    (6, 3, 32, 16, 5, [64, 4, 200], 1, False),
    (4, 2, 16, 32, 1, [90, 512, 513], 5, True),
    (8, 1, 128, 64, 1, [30000], 0, True),
    (8, 8, 64, 16, 1, [9001, 40], 4000, False),
    (2, 1, 64, 16, 40, [100, 41, 39], 0, False),
    (14, 2, 128, 16, 1, [333] * 20, 0, False),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("case", PAGED, ids=lambda c: "-".join(map(str, c[:5])) + f"-w{c[6]}-{sum(c[5])}")
def test_attention_matches_definition(P, case, codes, dtype):
    H, KH, hd, page, n, lens, window, with_sinks = case
    g, dt = gen(31), DT[dtype]
    pool = Pool(g, dt, codes, KH, hd, page, lens)
    q = rand(g, len(lens), n, H, hd, dtype=dt, scale=1.5)
    sinks = torch.randn(H, generator=g, device="cuda") if with_sinks else None
    want = paged_ref(pool, q, lens, window, sinks)
    got = P.attention_paged(q if n > 1 else q[:, 0], pool.k, pool.v, pool.tables, pool.lens, **pool.kw, window=window, sinks=sinks,
                            max_len=max(lens))
    check(got.view(q.shape), *want, codes)
    # without a bound of the lengths, one query as four dimensions
    got2 = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, window=window, sinks=sinks)
    check(got2, *want, codes)


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_attention_of_many_sequences(P, codes):
    """More sequences than one scan, long ones among short and empty ones."""
    rng, g = np.random.default_rng(5), gen(32)
    lens = [int(x) for x in rng.integers(0, 40, 700)]
    lens[3], lens[650] = 5000, 2100
    pool = Pool(g, torch.bfloat16, codes, 2, 64, 16, lens)
    q = rand(g, 700, 1, 8, 64, dtype=torch.bfloat16, scale=1.5)
    want = paged_ref(pool, q, lens)
    check(P.attention_paged(q[:, 0], pool.k, pool.v, pool.tables, pool.lens, **pool.kw)[:, None], *want, codes)
    short = pool.lens.clamp(max=50)                                # whole units: max_len says so
    pool.lens = short
    got = P.attention_paged(q[:, 0], pool.k, pool.v, pool.tables, short, **pool.kw, max_len=50)
    check(got[:, None], *paged_ref(pool, q, short.tolist()), codes)


def test_attention_of_scales_that_differ(P):
    """Values whose scales differ by 2^20 and more from block to block: the weights that meet them have a reference of their own."""
    for dtype in ("bf16", "fp16"):
        g, lens = gen(33), [900, 64, 17]
        pool = Pool(g, DT[dtype], True, 2, 128, 16, lens, spread=3.0)
        q = rand(g, 3, 2, 8, 128, dtype=DT[dtype], scale=1.5)
        check(P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw), *paged_ref(pool, q, lens), True)
    # and by more than fp32's weights hold: a block of 2^60 with little weight beside one of 2^-60 with all of it
    g = gen(34)
    pool = Pool(g, torch.bfloat16, True, 1, 64, 16, [32])
    page = pool.tables[0].tolist()
    pool.ks[:], pool.vs[page[0]], pool.vs[page[1]] = 2.0 ** -5, 2.0 ** 60, 2.0 ** -60
    pool.k[page[0]], pool.k[page[1]] = torch.tensor(-64.0, device="cuda").to(E4M3), torch.tensor(64.0, device="cuda").to(E4M3)
    q = torch.ones(1, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    want = paged_ref(pool, q, [32])
    check(P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw), *want, True)
    pool.vs[page[0]] = 2.0 ** -60                                  # all of it far below fp16's range
    want, a, delta = paged_ref(pool, q, [32])
    got = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw)
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * delta) * 1.05 * a).all())


def poison(pool, value):
    """Everything that lens does not reach, and pages of no sequence, in place."""
    used = torch.zeros(pool.n, pool.page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(pool.lens.tolist()):
        j = torch.arange(n, device="cuda")
        t = pool.tables[b].long()[j // pool.page]
        ok = (t >= 0) & (t < pool.n)
        used[t[ok], (j % pool.page)[ok]] = True
    for x in (pool.k, pool.v):
        if pool.codes:
            x.view(torch.uint8).transpose(1, 2)[~used] = 0x7f            # NaN, the only one of these that e4m3 has
        else:
            x.transpose(1, 2)[~used] = value
    if pool.codes:
        blocks = used.view(pool.n, -1, 16).any(2)
        for s in (pool.ks, pool.vs):
            s.transpose(1, 2)[~blocks] = math.nan


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("n", [1, 3])
def test_what_no_query_attends_to_may_hold_anything(P, n, codes, dtype):
    g, lens, dt = gen(35), [0, 3, 50, 16, 333, 700], DT[dtype]
    for hd in (64, 128):
        pool = Pool(g, dt, codes, 2, hd, 64, lens, spare=4)
        pool.tables[4, 2] = -1                                    # a page given back
        q = rand(g, len(lens), n, 8, hd, dtype=dt)
        call = lambda: P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw)  # noqa: E731
        clean = call()
        check(clean, *paged_ref(pool, q, lens), codes)
        for value in (math.nan, math.inf):
            poison(pool, value)
            assert torch.equal(call(), clean)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 8])
def test_values_that_some_queries_see(P, G, hd, codes, dtype):
    """A value that is not finite reaches the queries that attend to it, in its dimension, and no others: behind the causal edge and before the window."""
    g, n, KH, dt, window = gen(36), 6, 2, DT[dtype], 40
    pool = Pool(g, dt, codes, KH, hd, 16, [100])
    q = rand(g, 1, n, KH * G, hd, dtype=dt)
    call = lambda: P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, window=window)  # noqa: E731
    clean = call()
    bad = [(97, 3), (99, hd - 1), (57, 0), (59, hd // 2), (61, 1)]
    for j, d in bad:
        pool.v[int(pool.tables[0, j // 16]), 1, j % 16, d] = torch.tensor(math.nan, device="cuda").to(pool.v.dtype)
    got = call()
    want = torch.zeros(n, KH * G, hd, dtype=torch.bool, device="cuda")
    for j, d in bad:
        for i in range(n):
            e = 100 - n + i
            if e - window < j <= e:
                want[i, G:, d] = True
    assert torch.equal(torch.isnan(got[0]), want)
    # the others are as if these values were any numbers
    for j, d in bad:
        pool.v[int(pool.tables[0, j // 16]), 1, j % 16, d] = torch.tensor(0.0, device="cuda").to(pool.v.dtype)
    out, a, delta = paged_ref(pool, q, [100], window)
    check(torch.where(want, out[0].to(dt), got[0])[None], out, a, delta, codes)


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_scores_that_are_not_finite(P, codes):
    g, lens, KH = gen(37), [70, 70, 70, 300], 2
    pool = Pool(g, torch.bfloat16, codes, KH, 64, 16, lens)
    q = rand(g, 4, 1, 4, 64, dtype=torch.bfloat16)
    q[..., 0] = q[..., 0].abs() + 0.125
    clean = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw)
    at = lambda b, j: (int(pool.tables[b, j // 16]), 1, j % 16)  # noqa: E731
    pool.k[at(0, 33)] = torch.tensor(math.nan, device="cuda").to(pool.k.dtype)
    pool.k[at(3, 299)] = torch.tensor(math.nan, device="cuda").to(pool.k.dtype)
    q[1, 0, 2:, 5] = math.nan
    if not codes:
        k = pool.k[at(2, 40)]
        k[0] = -math.inf                                          # a score of -inf: no weight
        keep = torch.arange(70, device="cuda") != 40
        kk, vv = pool.values("k", 2, 70)[1][keep], pool.values("v", 2, 70)[1][keep]
        want = attend(q[2, 0, 2:], kk, vv, torch.ones(2, 69, dtype=torch.bool, device="cuda"), 1 / 8, None)
    got = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw)
    assert bool(torch.isnan(got[[0, 1, 3], 0, 2:]).all()) and torch.equal(got[:, :, :2], clean[:, :, :2])
    if codes:
        assert torch.equal(got[2], clean[2])
    else:
        check(got[2, 0, 2:], *want, codes)
        pool.k[at(2, 40)][0] = math.inf
        assert bool(torch.isnan(P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens)[2, 0, 2:]).all())


def test_weights_far_below_the_largest(P):
    """4,095 keys of 2^-20 of the largest weight beside one of no value: all of the output is theirs."""
    for dtype in ("bf16", "fp16"):
        for codes in (True, False):
            g, m = gen(38), 4096
            pool = Pool(g, DT[dtype], codes, 1, 64, 16, [m])
            pool.k[:], q = torch.zeros((), device="cuda").to(pool.k.dtype), torch.zeros(1, 1, 2, 64, dtype=DT[dtype], device="cuda")
            t, r = int(pool.tables[0, 100]), 7
            pool.k[t, 0, r, 0] = torch.tensor(20.0, device="cuda").to(pool.k.dtype)
            pool.v[t, 0, r] = torch.zeros((), device="cuda").to(pool.v.dtype)
            pool.v[:, :, :, :32] = pool.v[:, :, :, :32].float().abs().to(pool.v.dtype)
            if codes:
                pool.ks[:] = 1.0
            q[..., 0] = 1.0
            want = paged_ref(pool, q, [m], scale=math.log(2.0))
            check(P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, scale=math.log(2.0)), *want, codes)


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_attention_strided_views(P, codes):
    g, lens, KH = gen(39), [100, 37, 260], 2
    a = Pool(g, torch.float16, codes, KH, 64, 32, lens)
    y = rand(g, 3, 2, 12, 64, dtype=torch.float16)
    want = P.attention_paged(y[:, :, 2:10].contiguous(), a.k, a.v, a.tables, a.lens, **a.kw)
    k, v = (x.view(torch.uint8 if codes else torch.int16).transpose(1, 2).contiguous().transpose(1, 2).view(x.dtype) for x in (a.k, a.v))
    kw = {n: None if s is None else s.permute(1, 2, 0).contiguous().permute(2, 0, 1) for n, s in a.kw.items()}
    wide = torch.full((3, a.tables.shape[1] + 3), 999, dtype=torch.int32, device="cuda")
    wide[:, 1:1 + a.tables.shape[1]] = a.tables
    out = torch.full((8, 3, 2, 64), 5.0, dtype=torch.float16, device="cuda").permute(1, 2, 0, 3)
    got = P.attention_paged(y[:, :, 2:10], k, v, wide[:, 1:1 + a.tables.shape[1]], a.lens, **kw, out=out)
    assert got is out and torch.equal(got, want)
    # heads of one token each, rows of a wider tensor
    one = P.attention_paged(y[:, 1, 2:10], k, v, a.tables, a.lens, **kw)
    assert torch.equal(one, P.attention_paged(y[:, 1:, 2:10].contiguous(), a.k, a.v, a.tables, a.lens, **a.kw)[:, 0])


def test_lens_beyond_the_bounds(P):
    g = gen(40)
    pool = Pool(g, torch.bfloat16, True, 2, 64, 16, [64, 64, 64])
    q = rand(g, 3, 8, 64, dtype=torch.bfloat16)
    call = lambda lens, **kw: P.attention_paged(q, pool.k, pool.v, pool.tables, lens, **pool.kw, **kw)  # noqa: E731
    assert torch.equal(call(ints(64, 64, 0)), call(ints(65, 2147483647, -3)))
    assert torch.equal(call(ints(30, 20, 30)), call(ints(64, 20, 31), max_len=30))
    assert torch.equal(call(ints(30, 20, 30), window=2 ** 40), call(ints(30, 20, 30)))


def test_far_places(P):
    """Pools of more than 2^31 bytes and elements: the last pages."""
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 40 GB")
    g, KH, hd, page = gen(41), 4, 128, 256
    for codes, dt in ((True, torch.bfloat16), (False, torch.float16)):
        n = (1 << 31) // (KH * hd * page) + 40
        k, v = (torch.empty(n, KH, page, hd, dtype=E4M3 if codes else dt, device="cuda") for _ in range(2))
        s = [torch.empty(n, KH, page // 16, device="cuda") if codes else None for _ in range(2)]
        kw = {"k_scales": s[0], "v_scales": s[1]}
        tables, lens = ints(n - 1, n - 3, n - 2).view(1, 3), ints(700)
        kn, vn = (rand(g, 700, KH, hd, dtype=dt) for _ in range(2))
        P.cache_append(kn, vn, k, v, tables, lens, ints(0, 700), **kw)
        small, at = Pool(g, dt, codes, KH, hd, page, [700]), ints(2, 0, 1)
        small.tables, last = at.view(1, 3), slice(n - 3, n)
        small.n, small.k, small.v, small.ks, small.vs = 3, k[last].clone(), v[last].clone(), *(None if x is None else x[last].clone() for x in s)
        kb, vb = P.cache_gather(k, v, tables, ints(0, 700), 700, **kw, dtype=dt)
        assert torch.equal(kb, small.values("k", 0, 700).transpose(0, 1).to(dt)) and torch.equal(vb, small.values("v", 0, 700).transpose(0, 1).to(dt))
        assert float((kb.float() - kn.float()).abs().max()) <= (2.0 ** -4 * float(kn.float().abs().max()) if codes else 0.0)
        q = rand(g, 1, 32, hd, dtype=dt)
        assert torch.equal(P.attention_paged(q, k, v, tables, lens, **kw),
                           P.attention_paged(q, small.k, small.v, small.tables, lens, **small.kw))
        del k, v, s, kw
        torch.cuda.empty_cache()


# ---- how they are called

def test_streams_graphs_and_repeats(P):
    """Captured calls replayed with other lengths, two graphs in turn, a stream of its own: the same bits."""
    g, B, KH, hd, page = gen(42), 6, 4, 128, 16
    pool = Pool(g, torch.bfloat16, True, KH, hd, page, [900] * B)
    f = P.rotary_frequencies(hd, device="cuda")[0]
    q, k, v = (rand(g, B, h, hd, dtype=torch.bfloat16) for h in (32, KH, KH))
    lens = ints(5, 0, 900, 333, 16, 17)

    def step(p, n):
        y = P.cache_append(k, v, p.k, p.v, p.tables, n, **p.kw, freqs=f, q=q)
        o = P.attention_paged(y, p.k, p.v, p.tables, n, **p.kw)
        kb, vb = P.cache_gather(p.k, p.v, p.tables, torch.arange(B + 1, device="cuda").int() * 20, 20 * B, **p.kw)
        return y, o, kb, vb

    base, other = pool.clone(), ints(600, 1, 17, 0, 700, 32)
    want = step(pool.clone(), lens), step(pool.clone(), other)
    assert all(torch.equal(x, y) for x, y in zip(step(pool.clone(), lens), want[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(pool.clone(), lens)
        n, work = lens.clone(), [pool.clone(), pool.clone()]
        step(work[0], n)                                           # warm
        graphs, outs = [], []
        for p in work:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(step(p, n))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want[0]))
    for turn, values in enumerate((other, lens, other)):
        n.copy_(values)
        for p in work:
            for x in ("k", "v", "ks", "vs"):
                getattr(p, x).copy_(getattr(base, x))
        graphs[0].replay()
        graphs[1].replay()
        graphs[1].replay()                                         # appending the same once more changes nothing
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(x, y) for x, y in zip(o, want[turn % 2 == 0]))


def test_empty_calls(P):
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    f, i = z(32, dt=torch.float64), lambda *s: z(*s, dt=torch.int32)
    pages = z(3, 2, 16, 64)
    assert P.rotary(z(0, 4, 64), z(0, 2, 64), i(0), f)[1].shape == (0, 2, 64)
    assert P.cache_append(z(0, 2, 64), z(0, 2, 64), pages, pages, i(0, 4), i(0), q=z(0, 4, 64)).shape == (0, 4, 64)
    P.cache_append(z(2, 2, 64) + 1, z(2, 2, 64) + 1, pages, pages, i(2, 0), i(2) + 5)        # tables without columns
    assert not bool(pages.any())
    assert P.attention_paged(z(0, 4, 64), pages, pages, i(0, 4), i(0)).shape == (0, 4, 64)
    assert P.attention_paged(z(2, 0, 4, 64), pages, pages, i(2, 4), i(2) + 3).shape == (2, 0, 4, 64)
    none = z(0, 2, 16, 64)
    for p, t in ((pages, i(2, 0)), (none, i(2, 3))):                # no columns, no pages: no keys
        assert not bool(P.attention_paged(z(2, 4, 64) + 1, p, p, t, i(2) + 9).any())
        k, v = P.cache_gather(p, p, t, ints(0, 3, 5), 5)
        assert not bool(k.any()) and not bool(v.any())
    assert P.cache_gather(pages, pages, i(2, 4), i(3), 0)[0].shape == (0, 2, 64)
    assert P.cache_gather(pages, pages, i(0, 4), i(1), 0)[0].shape == (0, 2, 64)


def test_refusals(P, gpu):
    bf, dev = torch.bfloat16, "cuda"
    z = lambda *s, dt=bf: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
    q, k, f, i = z(4, 4, 64), z(4, 2, 64), z(32, dt=torch.float64), ints(1, 2, 3, 4)
    pages, codes, scales, tables = z(3, 2, 32, 64), z(3, 2, 32, 64, dt=E4M3), z(3, 2, 2, dt=torch.float32), z(4, 2, dt=torch.int32)

    def no(text, fn, *args, **kw):
        with pytest.raises(ValueError, match=text):
            fn(*args, **kw)

    R = P.rotary
    no("CUDA tensor", R, q, k, i.cpu(), f)
    no("bfloat16 or float16", R, q.float(), k.float(), i, f)
    no("k must be bfloat16", R, q, k.half(), i, f)
    no("do not fit", R, q, k[:3], i, f)
    no("int32", R, q, k, i.long(), f)
    no("float64", R, q, k, i, f.float())
    no("frequencies", R, q, k, i, z(33, dt=torch.float64))
    no("q_norm", R, q, k, i, f, q_norm=z(63, dt=torch.float32))
    no("contiguous", R, q.transpose(1, 2).contiguous().transpose(1, 2), k, i, f)
    no("strides", R, z(4, 4, 68)[..., :64], k, i, f)
    no("out", R, q, k, i, f, out=(q, None))
    no("out", R, q, None, i, f, out=(q, k))
    no("out", R, q, k, i, f, out=q)
    no("eps", R, q, k, i, f, eps=-1.0)
    no("amplitude", R, q, k, i, f, amplitude=math.nan)
    no("strides", R, q, k, i, f, out=(z(1, 4, 64).expand(4, 4, 64), k))
    A = P.cache_append
    no("do not fit", A, k, k[:3], pages, pages, tables, i)
    no("as many tokens", A, k, k, pages, pages, tables[:3], i[:3])
    no("k_pages must be bfloat16 or float8_e4m3fn", A, k, k, pages.half(), pages.half(), tables, i)
    no("v_pages", A, k, k, pages, codes, tables, i)
    no("have no scales", A, k, k, pages, pages, tables, i, k_scales=scales, v_scales=scales)
    no("need k_scales", A, k, k, codes, codes, tables, i, k_scales=scales)
    no("v_scales", A, k, k, codes, codes, tables, i, k_scales=scales, v_scales=scales[:, :, :1])
    no("page must be", A, k, k, pages[:, :, :24], pages[:, :, :24], tables, i)
    no("cu", A, k, k, pages, pages, tables, i, i[:3])
    no("lens", A, k, k, pages, pages, tables, i[None])
    no("tables", A, k, k, pages, pages, tables[0], i)
    no("out is for q", A, k, k, pages, pages, tables, i, out=q)
    no("out", A, k, k, pages, pages, tables, i, q=q, out=q[:, :2])
    no("positions", A, k, k, pages, pages, tables, i, positions=i[:2])
    no("strides of pages", A, k, k, pages[:1].expand(3, 2, 32, 64), pages, tables, i)
    no("multiple of 16", A, *(z(4, 2, 72) for _ in range(2)), *(z(3, 2, 32, 72, dt=E4M3) for _ in range(2)), tables, i, k_scales=scales,
       v_scales=scales)
    T = P.attention_paged
    no("do not fit", T, q[:3], pages, pages, tables, i)
    no("multiple of n_kv_heads", T, q[:, :3], pages, pages, tables, i)
    no("need k_scales", T, q, codes, codes, tables, i)
    no("sinks", T, q, pages, pages, tables, i, sinks=z(2, dt=torch.float32))
    no("window", T, q, pages, pages, tables, i, window=-1)
    no("scale must", T, q, pages, pages, tables, i, scale=0.0)
    no("negative", T, q, pages, pages, tables, i, max_len=-1)
    no("out", T, q, pages, pages, tables, i, out=q[:2])
    no("at most 128", T, *(x for x in (z(4, 4, 136), z(3, 2, 32, 136), z(3, 2, 32, 136))), tables, i)
    G = P.cache_gather
    no("total", G, pages, pages, tables, ends([1] * 4), -1)
    no("are not read as", G, pages, pages, tables, ends([1] * 4), 4, dtype=torch.float16)
    no("bfloat16 or float16", G, codes, codes, tables, ends([1] * 4), 4, k_scales=scales, v_scales=scales, dtype=torch.float32)
    no("cu", G, pages, pages, tables, ends([1] * 3), 3)
    no(r"out\[1\]", G, pages, pages, tables, ends([1] * 4), 4, out=(k, k[:3]))
    for t in (q, k, f, pages, scales):
        t.requires_grad_(True)
        with pytest.raises(ValueError, match="backward"):
            if t is q:
                T(q, pages, pages, tables, i)
            elif t is scales:
                G(codes, codes, tables, ends([1] * 4), 4, k_scales=scales, v_scales=scales)
            elif t is pages:
                G(pages, pages, tables, ends([1] * 4), 4)
            elif t is k:
                A(k, k.detach(), pages, pages, tables, i)
            else:
                R(q.detach(), None, i, f)
        with torch.no_grad():
            R(q, k, i, f)
        t.requires_grad_(False)
    # host memory and small workspaces at the C entries
    h, d, st = np.zeros(4096, np.float32).ctypes.data, z(1 << 16).data_ptr(), (ctypes.c_int64 * 21)(*[64] * 21)
    assert gpu.tg_rotary(0, h, None, d, None, d, d, None, None, 1, 1, 0, 64, 32, 0, 1.0, 0.0, st, None) == 3
    assert "device memory" in tg.last_error(gpu)[1]
    assert gpu.tg_attention_paged(0, 16, d, d, d, None, None, d, d, d, None, 8, 1, 2, 16, 999, 10000, 1, 1, 64, st, 0, 0.125, None, 0, None) == 3
    assert "workspace" in tg.last_error(gpu)[1]
    versions = pages._version, scales._version
    A(k, k, pages, pages.clone(), tables, ints(1, 0, 0, 0))
    A(k, k, codes, codes.clone(), tables, ints(1, 0, 0, 0), k_scales=scales, v_scales=scales.clone())
    assert pages._version > versions[0] and scales._version > versions[1]


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_a_batch_from_prompts_to_drafts(P, codes):
    """Prompts in chunks, next tokens, drafts of which some are dropped, pages behind the window given back: every step's attention
    against what the cache holds, and the cache at the end against the tokens."""
    from tinygiant_b200 import attention as A
    g, H, KH, hd, page, dt = gen(43), 8, 2, 64, 16, torch.bfloat16
    B, lens = 3, [0, 0, 0]
    pool = Pool(g, dt, codes, KH, hd, page, [300] * B)
    f, amp = P.rotary_frequencies(hd, 150000.0, scaling="yarn", factor=8, original_len=64, device="cuda")
    w = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)]
    kept = [[] for _ in range(B)]                                  # k and v of each token as they came

    def append(new):
        for b in range(B):
            lens[b] += new[b]
        pool.lens = ints(*lens)
        T = sum(new)
        q, k, v = (rand(g, T, h, hd, dtype=dt) for h in (H, KH, KH))
        at = 0
        for b in range(B):
            kept[b] += list(zip(k[at:at + new[b]], v[at:at + new[b]]))
            at += new[b]
        return P.cache_append(k, v, pool.k, pool.v, pool.tables, pool.lens, ends(new), **pool.kw, freqs=f, amplitude=amp, q=q,
                              q_norm=w[0], k_norm=w[1])

    for new in ([33, 1, 100], [60, 20, 0], [7, 130, 16]):          # chunks of prompts
        q = append(new)
        cu = ends(lens)
        k, v = P.cache_gather(pool.k, pool.v, pool.tables, cu, sum(lens), **pool.kw)
        o = A.attention_prompt(q, k, v, ends(new), cu)
        for b in range(B):
            if new[b]:
                rows = slice(sum(new[:b]), sum(new[:b + 1]))
                view = pool.clone()
                view.tables, view.lens = pool.tables[b:b + 1], pool.lens[b:b + 1]
                check(o[None, rows], *paged_ref(view, q[None, rows], lens[b:b + 1]), False)
    for n, keep in ((1, 1), (1, 1), (4, 2), (1, 1), (4, 1), (3, 3), (1, 1)):      # tokens; drafts, the first `keep` of which stay
        q = append([n] * B).view(B, n, H, hd)
        got = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, window=50)
        check(got, *paged_ref(pool, q, lens, 50), codes)
        for b in range(B):
            lens[b] -= n - keep
            del kept[b][len(kept[b]) - (n - keep):]
    for b in range(B):
        k, v = (torch.stack(x) for x in zip(*kept[b]))
        k64, d = rotate64(k, torch.arange(lens[b], device="cuda"), f, False, amp, w[1])
        for x, want, e in (("k", k64, d), ("v", v.double(), torch.zeros_like(k64))):
            got = pool.values(x, b, lens[b]).transpose(0, 1)
            if not codes:
                near(got.to(dt), want, e)
                continue
            s = (pool.ks if x == "k" else pool.vs)[pool.tables[b].long()].double()        # [columns, KH, 1] of pages of one block
            s = s[torch.arange(lens[b], device="cuda") // 16]
            # rounded again as its block's scale grew, each time by half of the least step at most below what it had lost before
            tol = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * s) + 2.0 ** -9 * s + e * (1 + 2.0 ** -4)
            assert bool(((got - want).abs() <= tol).all())
    # pages that lie behind the window altogether are given back
    pool.lens = ints(*lens)
    q = rand(g, B, H, hd, dtype=dt)
    before = P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, window=50)
    for b in range(B):
        pool.tables[b, :(lens[b] - 50) // page] = -1
    assert torch.equal(P.attention_paged(q, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, window=50), before)


@pytest.mark.parametrize("bits,window", [("8", "0"), ("16", "0"), ("8", "200")])
def test_serving_example(gpu, bits, window):
    """Prompts in chunks, drafts, pages given back and the experts' steps through examples/serve_paged.py, the last attention checked."""
    import importlib.util
    from pathlib import Path
    spec = importlib.util.spec_from_file_location("serve_paged", Path(__file__).resolve().parents[1] / "examples" / "serve_paged.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(["--batch", "3", "--chunk", "200", "--steps", "12", "--page", "32", "--bits", bits, "--window", window]) < 2e-2


# heads, kv heads, head_dim: two and three rows of a thread, in one share of a token's rows and in several
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("H,KH,hd", [(8, 2, 64), (32, 4, 128), (40, 4, 128), (140, 4, 96), (0, 2, 128)])
def test_many_tokens_equal_few_at_a_time(P, H, KH, hd, codes, norms):
    """Thousands of tokens in one call give the bits of calls that each hold a token or two of a CTA."""
    g, T, step = gen(31), 2803, 160
    pool = Pool(g, torch.bfloat16, codes, KH, hd, 32, [T + 48])
    few = pool.clone()
    q, k, v = rand(g, T, H + 2 * KH, hd, dtype=torch.bfloat16, scale=3.0).split([H, KH, KH], 1)
    w = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") if norms else None for _ in range(2)]
    kw = {"freqs": P.rotary_frequencies(hd, device="cuda")[0], "q_norm": w[0] if H else None, "k_norm": w[1]}
    out = P.cache_append(k, v, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, **kw, q=q if H else None)
    pos = torch.arange(48, T + 48, device="cuda").int()
    turned = P.rotary(q, k, pos, **kw) if H else P.rotary(k, None, pos, kw["freqs"], q_norm=w[1])[::-1]
    assert not H or torch.equal(out, turned[0])
    for a in range(0, T, step):
        b = min(T, a + step)
        y = P.cache_append(k[a:b], v[a:b], few.k, few.v, few.tables, ints(b + 48), **few.kw, **kw, q=q[a:b] if H else None)
        z = P.rotary(k[a:b], None, pos[a:b], kw["freqs"], q_norm=w[1])[0]
        assert (not H or torch.equal(y, out[a:b])) and torch.equal(z, turned[1][a:b])
    assert torch.equal(bits(pool.k), bits(few.k)) and torch.equal(bits(pool.v), bits(few.v))
    assert not codes or (torch.equal(pool.ks, few.ks) and torch.equal(pool.vs, few.vs))
    if not codes:
        row = (pool.tables[0].long()[pos.long() // 32], pos.long() % 32)
        assert torch.equal(pool.k.transpose(1, 2)[row], turned[1]) and torch.equal(pool.v.transpose(1, 2)[row], v)


@pytest.mark.parametrize("codes", [True, False], ids=["8bit", "16bit"])
def test_more_sequences_than_a_cta_keeps_offsets_of(P, codes):
    """1,500 sequences of none to three new tokens, in one call and in two; and read back."""
    g, B, KH, hd = gen(32), 1500, 2, 64
    new = [(7 * b) % 4 for b in range(B)]
    lens = [16 * (b % 3) + n for b, n in enumerate(new)]
    pool = Pool(g, torch.bfloat16, codes, KH, hd, 16, lens)
    two, T, half = pool.clone(), sum(new), sum(new[:B // 2])
    k, v = rand(g, T, KH, hd, dtype=torch.bfloat16), rand(g, T, KH, hd, dtype=torch.bfloat16)
    f = P.rotary_frequencies(hd, device="cuda")[0]
    P.cache_append(k, v, pool.k, pool.v, pool.tables, pool.lens, ends(new), **pool.kw, freqs=f)
    for rows, seqs in ((slice(0, half), slice(0, B // 2)), (slice(half, T), slice(B // 2, B))):
        P.cache_append(k[rows], v[rows], two.k, two.v, two.tables[seqs], two.lens[seqs], ends(new[seqs]), **two.kw, freqs=f)
    assert torch.equal(bits(pool.k), bits(two.k)) and torch.equal(bits(pool.v), bits(two.v))
    keys, vals = P.cache_gather(pool.k, pool.v, pool.tables, ends(lens), sum(lens), **pool.kw)
    at = [0, *np.cumsum(lens).tolist()]
    for b in range(0, B, 97):
        assert torch.equal(keys[at[b]:at[b + 1]].double(), pool.values("k", b, lens[b]).transpose(0, 1).to(torch.bfloat16).double())
        assert torch.equal(vals[at[b]:at[b + 1]].double(), pool.values("v", b, lens[b]).transpose(0, 1).to(torch.bfloat16).double())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd,n,inter,norm", [(128, 64, False, True), (64, 32, True, False), (80, 20, False, True), (96, 47, False, False), (128, 0, False, True)])
def test_codes_are_the_exact_values_rounded(P, hd, n, inter, norm, dtype):
    """Hundreds of thousands of codes of normed and rotated keys: the 64-bit values' nearest, none decided by fp32's rounding."""
    g, T, KH = gen(41), 1024, 4
    pool = Pool(g, DT[dtype], True, KH, hd, 64, [T])
    k = rand(g, T, KH, hd, dtype=DT[dtype], scale=2.0)
    f = P.rotary_frequencies(2 * n, 1e6, device="cuda")[0] if n else None
    w = 1 + 0.3 * torch.randn(hd, generator=g, device="cuda") if norm else None
    P.cache_append(k, k, pool.k, pool.v, pool.tables, pool.lens, **pool.kw, freqs=f, interleaved=inter, k_norm=w)
    want, _ = rotate64(k, torch.arange(T, device="cuda"), f, inter, 1.0, w)
    scale, _ = P.cache_gather(torch.ones_like(pool.k.float()).to(E4M3), pool.v, pool.tables, ints(0, T), T, k_scales=pool.ks, v_scales=pool.vs,
                              dtype=torch.bfloat16)
    y = want / scale.double()
    y32 = y.float()
    short = torch.where(y32.double().abs() > y.abs(), torch.nextafter(y32, torch.zeros_like(y32)), y32)      # towards zero
    odd = torch.where(short.double() == y, short.view(torch.int32), short.view(torch.int32) | 1).view(torch.float32)
    p = torch.arange(T, device="cuda")
    codes = pool.k.transpose(1, 2)[pool.tables[0].long()[p // 64], p % 64]
    assert torch.equal(bits(codes), bits(odd.to(E4M3)))
