"""Attention operators where the numbers or the calls are unusual: scores
that are not finite, weights far below the row's largest, windows beyond any
position, prefix values that are not finite under many window edges.

Tolerances are those of test_gpu_attn_ops.  A weight of 2^-24 of its row's
largest or more is a normal number in either 16-bit type, so its rounding is
the unit roundoff u that the tolerance has; at 2^-24.5 it is at most 1.5 u, and
what the tolerance leaves for the scores (0.6 u at least there) covers that.
"""
import math

import pytest

import tinygiant_b200 as tg
from test_gpu_attn_ops import DT, attend, check, ends, gen, prompt_ref, rand, shared_ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def A(gpu):
    from tinygiant_b200 import attention
    return attention


# ---- scores that are not finite: the definition's softmax is NaN for a row
# that attends to a score of NaN or +inf, and gives a key of -inf no weight.
# 32 key heads hold one odd key each, at every place among 32, in a block of
# keys that later rows see whole.

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_prompt_scores_that_are_not_finite(A, poison, hd, dtype):
    g, dt, n, KH, H = gen(51), DT[dtype], 420, 32, 64
    q = rand(g, n, H, hd, dtype=dt)
    q[..., 0] = q[..., 0].abs() + 0.125                       # an infinity keeps its sign
    k, v = (rand(g, n, KH, hd, dtype=dt) for _ in range(2))
    clean = A.attention_prompt(q, k, v, ends([n]))
    at = 128 + 32 + torch.arange(KH, device="cuda")
    k[at, torch.arange(KH, device="cuda"), 0] = poison
    got = A.attention_prompt(q, k, v, ends([n]))
    sees = (torch.arange(n, device="cuda")[:, None] >= at).repeat_interleave(2, 1)      # [n, H]
    assert torch.equal(got[~sees], clean[~sees])
    if poison == -math.inf:                                   # as if the key were not there
        for kh in (0, 1, 7, 14, 15, 30, 31):
            rest = torch.arange(n, device="cuda") != at[kh]
            for h in (2 * kh, 2 * kh + 1):
                i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")
                kk = torch.where(rest[:, None], k[:, kh], 0.0)
                o, _, a, d = attend(q[:, h], kk, v[:, kh], (j <= i) & rest, hd ** -0.5, None)
                check(got[:, h], o, a, d)
        assert not bool(torch.isnan(got).any())
    else:
        assert bool(torch.isnan(got[sees]).all()), int((~torch.isnan(got[sees])).any(-1).sum())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_prefix_scores_that_are_not_finite(A, poison, hd, dtype):
    g, dt, P, KH, H, lens = gen(52), DT[dtype], 384, 32, 64, [9, 0, 40]
    q = rand(g, 3, H, hd, dtype=dt)
    q[..., 0] = q[..., 0].abs() + 0.125
    pk, pv = (rand(g, KH, P, hd, dtype=dt) for _ in range(2))
    k, v = (rand(g, 3, KH, 40, hd, dtype=dt) for _ in range(2))
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    heads = torch.arange(KH, device="cuda")
    pk[heads, 128 + 64 + heads, 0] = poison
    w = torch.zeros(3, KH, 40, device="cuda")
    got = A.attention_shared(q, pk, pv, k, v, n, weights=w)
    if poison == -math.inf:
        keep = torch.stack([torch.cat([torch.arange(192 + h), torch.arange(193 + h, P)]) for h in range(KH)]).cuda()
        at = keep[..., None].expand(KH, P - 1, hd)
        out, a, delta, ww, wd = shared_ref(q, torch.gather(pk, 1, at), torch.gather(pv, 1, at), k, v, lens, 0, None, hd ** -0.5)
        check(got, out, a, delta)
        assert bool(((w.double() - ww).abs() <= 1.05 * wd + ww * 2.0 ** -22).all())
    else:
        assert bool(torch.isnan(got).all()), int((~torch.isnan(got)).sum())
        there = torch.arange(40, device="cuda") < n[:, None]
        assert bool(torch.isnan(w.transpose(1, 2)[there]).all()) and not bool(w.transpose(1, 2)[~there].any())


@pytest.mark.parametrize("hd", [64, 128])
def test_rows_whose_scores_are_all_minus_infinity(A, hd):
    """No key has any weight: zeros, as for a row without a key; a later finite score takes everything."""
    g, n, H, KH = gen(53), 600, 4, 2
    q, k, v = rand(g, n, H, hd, dtype=torch.bfloat16), *(rand(g, n, KH, hd, dtype=torch.bfloat16) for _ in range(2))
    q[..., 0] = 1
    k[:, 0, 0] = -math.inf
    k[:400, 1, 0] = -math.inf
    got = A.attention_prompt(q, k, v, ends([n]))
    assert not bool(got[:, :2].any()) and not bool(got[:400, 2:].any())
    check(got[400:, 2:], *prompt_ref(q[400:, 2:], k[400:, 1:], v[400:, 1:], [200], [200], 0, None, hd ** -0.5))
    sinks = torch.zeros(H, device="cuda")
    assert not bool(A.attention_prompt(q, k, v, ends([n]), sinks=sinks)[:, :2].any())
    pk, pv = k.transpose(0, 1).contiguous(), v.transpose(0, 1).contiguous()
    c = torch.zeros(2, KH, 8, hd, dtype=torch.bfloat16, device="cuda")
    got = A.attention_shared(q[:2], pk[:, :384], pv[:, :384], c, c, torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert not bool(got.any())


@pytest.mark.parametrize("hd", [64, 128])
def test_a_query_that_is_not_finite_stays_in_its_row(A, hd):
    g, n, H, KH = gen(54), 700, 4, 2
    q, k, v = rand(g, n, H, hd, dtype=torch.bfloat16), *(rand(g, n, KH, hd, dtype=torch.bfloat16) for _ in range(2))
    clean = A.attention_prompt(q, k, v, ends([n]))
    q[5, 1, 3], q[333, 2, 0], q[699, 0, 1] = math.nan, math.inf, -math.inf
    got = A.attention_prompt(q, k, v, ends([n]))
    bad = torch.zeros(n, H, dtype=torch.bool, device="cuda")
    bad[5, 1] = bad[333, 2] = bad[699, 0] = True
    assert torch.equal(got[~bad], clean[~bad]) and bool(torch.isnan(got[bad]).all())


# ---- values that are not finite in more partly seen blocks than a unit notes

@pytest.mark.parametrize("poison", [math.inf, math.nan])
def test_prefix_values_under_many_window_edges(A, poison):
    """Sequences whose windows begin all over the prefix, an odd value in each block: those that see it get it."""
    g, dt, H, KH, hd, P, cap, window = gen(55), torch.bfloat16, 16, 16, 64, 4000, 2048, 4100
    lens = [100, 1999, 400, 700, 1000, 1300, 1600, 1900]      # first keys seen: len - 100
    q = rand(g, 8, H, hd, dtype=dt)
    pk, pv = (rand(g, KH, P, hd, dtype=dt) for _ in range(2))
    k, v = (rand(g, 8, KH, cap, hd, dtype=dt) for _ in range(2))
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    clean = A.attention_shared(q, pk, pv, k, v, n, window=window)
    at = list(range(60, 2000, 64))                            # two in every block that some see in part
    for i, j in enumerate(at):
        pv[3, j, i] = poison
    got = A.attention_shared(q, pk, pv, k, v, n, window=window)
    want = clean.clone()
    for i, j in enumerate(at):
        for b, m in enumerate(lens):
            if j >= P + m - window:
                want[b, 3, i] = poison
    same = (got == want) | (torch.isnan(got) & (torch.isnan(want) | torch.isinf(want)))   # 0 times infinity may be NaN
    assert bool(same.all()), int((~same).sum())


# ---- weights far below the largest that together matter

def rare_heavy(g, n, KH, hd, dt, low):
    """Keys with a score of 0 and no value at every 32nd place, the others at `low` with values about 1000."""
    k = torch.zeros(n, KH, hd, device="cuda")
    k[..., 0] = low
    v = 1000 + 50 * torch.randn(n, KH, hd, generator=g, device="cuda")
    k[::32, :, 0] = 0
    v[::32] = 0
    return k.to(dt), v.to(dt)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("low", [-12, -17])
def test_weights_far_below_the_largest(A, low, hd, dtype):
    """exp(-17) = 2^-24.5: below what an fp16 number resolves beside 1, yet all of the output."""
    g, dt, n, H, KH = gen(56), DT[dtype], 6400, 4, 2
    k, v = rare_heavy(g, n, KH, hd, dt, low)
    q = torch.zeros(8, H, hd, device="cuda")
    q[..., 0] = 1
    q = q.to(dt)
    check(A.attention_prompt(q, k, v, ends([8]), ends([n]), scale=1.0), *prompt_ref(q, k, v, [8], [n], 0, None, 1.0))
    sinks = torch.tensor([-math.inf, 0.0, 3.0, -20.0], device="cuda")
    got = A.attention_prompt(q, k, v, ends([8]), ends([n]), scale=1.0, sinks=sinks)
    check(got, *prompt_ref(q, k, v, [8], [n], 0, sinks, 1.0))
    kh, vh = k.transpose(0, 1)[None].expand(2, KH, n, hd).contiguous(), v.transpose(0, 1)[None].expand(2, KH, n, hd).contiguous()
    lens = [n, 3201]
    nn = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for pk, pv in ((None, None), (kh[0, :, :3200].contiguous(), vh[0, :, :3200].contiguous())):
        w = torch.zeros(2, KH, n, device="cuda")
        out, a, delta, ww, wd = shared_ref(q[:2], pk, pv, kh, vh, lens, 0, sinks, 1.0)
        check(A.attention_shared(q[:2], pk, pv, kh, vh, nn, scale=1.0, sinks=sinks, weights=w), out, a, delta)
        assert bool(((w.double() - ww).abs() <= 1.05 * wd + ww * 2.0 ** -22).all())
    out, a, delta, _, _ = shared_ref(q[:2], pk, pv, kh, vh, [0, 0], 0, None, 1.0)
    check(A.attention_shared(q[:2], pk, pv, kh, vh, nn * 0, scale=1.0), out, a, delta)


# ---- windows beyond any position

@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 40])
def test_windows_beyond_any_position(A, window):
    """They are no window, also where queries precede the first key."""
    g, dt = gen(57), torch.bfloat16
    q, k, v = rand(g, 40, 4, 64, dtype=dt), *(rand(g, 20, 2, 64, dtype=dt) for _ in range(2))
    want = A.attention_prompt(q, k, v, ends([40]), ends([20]))
    check(want, *prompt_ref(q, k, v, [40], [20], 0, None, 1 / 8))
    assert torch.equal(A.attention_prompt(q, k, v, ends([40]), ends([20]), window=window), want)
    c, n = rand(g, 4, 2, 8, 64, dtype=dt), torch.tensor([8, 0, 3, 5], dtype=torch.int32, device="cuda")
    p = rand(g, 2, 300, 64, dtype=dt)
    check(A.attention_shared(q[:4], p, p, c, c, n, window=window), *shared_ref(q[:4], p, p, c, c, [8, 0, 3, 5], 0, None, 1 / 8)[:3])


def test_windows_below_zero_are_refused(A):
    q, c = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16, device="cuda")
    for window in (-1, -2 ** 31, -2 ** 32, 1 - 2 ** 32):
        with pytest.raises(ValueError, match="window"):
            A.attention_prompt(q, c[:, :, 0], c[:, :, 0], ends([4]), window=window)
        with pytest.raises(ValueError, match="window"):
            A.attention_shared(q, None, None, c, c, ends([1] * 3), window=window)


# ---- evictions of caches of different lengths at the same time

def evict_args(cap, keep):
    g = gen(58)
    k = rand(g, 1, 1, cap, 8, dtype=torch.bfloat16)
    return k, k, torch.rand(1, 1, cap, generator=g, device="cuda"), torch.tensor([cap], dtype=torch.int32, device="cuda"), keep, 3


def test_a_shorter_eviction_leaves_a_captured_longer_one(A):
    """A smaller cache's call between the capture of a larger one's and its instantiation."""
    big, small = evict_args(40000, 100), evict_args(9000, 50)
    want, less = A.cache_evict(*big), A.cache_evict(*small)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = A.cache_evict(*big)
        got2 = A.cache_evict(*small)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and all(torch.equal(x, y) for x, y in zip(got2, less))


def test_evictions_from_two_threads(gpu):
    """Long and short caches cut down at the same time, many times, through the C entry (Python leaves its lock meanwhile)."""
    import ctypes
    import threading
    refused = []

    def args_of(cap, stream):
        k, _, w, n, keep, recent = evict_args(cap, 64)
        outs = [torch.zeros(keep * 8, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        outs += [torch.zeros(keep, device="cuda"), *(torch.zeros(m, dtype=torch.int32, device="cuda") for m in (1, keep))]
        strides = (ctypes.c_int64 * 8)(cap * 8, cap * 8, 8, cap * 8, cap * 8, 8, cap, cap)
        return (k, w, n, outs, strides), (k.data_ptr(), k.data_ptr(), w.data_ptr(), n.data_ptr(), *(x.data_ptr() for x in outs), 1, cap, 1,
                                          8, ctypes.addressof(strides), keep, recent, stream.cuda_stream)

    def loop(args):
        for _ in range(30000):
            if gpu.tg_cache_evict(*args):
                refused.append(tg.last_error(gpu))
                return

    keep, args = zip(*(args_of(cap, torch.cuda.Stream()) for cap in (40000, 9000)))
    torch.cuda.synchronize()
    threads = [threading.Thread(target=loop, args=(a,)) for a in args]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused, refused
    del keep


# ---- what tg_cuda_synchronize waits for

def test_synchronize_waits_for_the_librarys_stream_alone(A, gpu):
    """Work on the default stream goes on."""
    q, k = torch.ones(4, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    A.attention_prompt(q, k, k, ends([4]))
    gpu.tg_cuda_set_stream(None)
    assert gpu.tg_cuda_synchronize() == 0
    torch.cuda.synchronize()
    torch.cuda._sleep(1_000_000_000)                          # half a second on the legacy default stream
    done = torch.cuda.Event()
    done.record()
    assert gpu.tg_cuda_synchronize() == 0
    assert not done.query()
    torch.cuda.synchronize()


FIRST = """
import sys
sys.path.insert(0, {root!r})
import torch
from tinygiant_b200 import attention as A
bf = torch.bfloat16
q, k = torch.ones(3, 4, 64, dtype=bf, device="cuda"), torch.ones(3, 2, 64, dtype=bf, device="cuda")
cu = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
c, n = torch.ones(3, 2, 600, 64, dtype=bf, device="cuda"), torch.tensor([600, 1, 5], dtype=torch.int32, device="cuda")
w = torch.zeros(3, 2, 600, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = A.attention_prompt(q, k, k, cu)
    b = A.attention_shared(q, c[0], c[0], c, c, n, weights=w)
    e = A.cache_evict(c, c, w, n, 40, 4)
g.replay()
torch.cuda.synchronize()
assert bool((a == 1).all()) and bool((b == 1).all()) and e[3].tolist() == [40, 1, 5]
"""


def test_first_calls_of_a_process_can_be_captured(gpu):
    import subprocess
    import sys
    from pathlib import Path
    code = FIRST.format(root=str(Path(__file__).resolve().parents[1]))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ---- arguments that are no tensors

def test_arguments_that_are_no_tensors_are_value_errors(A):
    bf, cu = torch.bfloat16, ends([4])
    q, k = torch.zeros(4, 4, 64, dtype=bf, device="cuda"), torch.zeros(4, 2, 64, dtype=bf, device="cuda")
    c, n, w = torch.zeros(4, 2, 8, 64, dtype=bf, device="cuda"), ends([1] * 3), torch.zeros(4, 2, 8, device="cuda")

    def no(text, fn, *args, **kw):
        with pytest.raises(ValueError, match=text):
            fn(*args, **kw)

    P, S, E = A.attention_prompt, A.attention_shared, A.cache_evict
    no("q must", P, None, k, k, cu)
    no("k must", P, q, None, k, cu)
    no("v must", P, q, k, None, cu)
    no("cu_q", P, q, k, k, [0, 4])
    no("cu_k", P, q, k, k, cu, [0, 4])
    no("sinks", P, q, k, k, cu, sinks=[0.0] * 4)
    no("out must", P, q, k, k, cu, out=7)
    no("k must have 3", P, q, c, c, cu)
    no("k must have 4", S, q, None, None, k[:, 0], k[:, 0], n)
    no("v must", S, q, None, None, c, None, n)
    no("lens", S, q, None, None, c, c, [1] * 4)
    no("lens", S, q, None, None, c, c, None)
    no("lens", S, q[:1], None, None, c[:1], c[:1], n[0])
    no("prefix", S, q, 1, 1, c, c, n)
    no("weights", S, q, None, None, c, c, n, weights=[1.0])
    no("sinks", S, q, None, None, c, c, n, sinks=0.5)
    no("out must", S, q, None, None, c, c, n, out="out")
    no("k must", E, None, c, w, n, 4, 1)
    no("v must", E, c, None, w, n, 4, 1)
    no("weights", E, c, c, None, n, 4, 1)
    no("lens", E, c, c, w, None, 4, 1)
    no("CUDA tensor", E, c.cpu(), c.cpu(), w.cpu(), n.cpu(), 4, 1)


# ---- gradients

def test_gradients_are_refused_and_writes_in_place_are_counted(A):
    """The operators have no backward pass: where one would be recorded they say so."""
    bf, cu = torch.bfloat16, ends([4])
    q, k = torch.ones(4, 4, 64, dtype=bf, device="cuda"), torch.ones(4, 2, 64, dtype=bf, device="cuda")
    c, n, w = torch.ones(4, 2, 8, 64, dtype=bf, device="cuda"), ends([1] * 3), torch.zeros(4, 2, 8, device="cuda")
    sinks = torch.zeros(4, device="cuda", requires_grad=True)
    for i in range(3):
        args = [q, k, k]
        args[i] = args[i].clone().requires_grad_()
        with pytest.raises(ValueError, match="no backward"):
            A.attention_prompt(*args, cu)
        with torch.no_grad():
            assert bool((A.attention_prompt(*args, cu) == 1).all())
        args = [q, c, c]
        args[i] = args[i].clone().requires_grad_()
        with pytest.raises(ValueError, match="no backward"):
            A.attention_shared(args[0], None, None, args[1], args[2], n)
    with pytest.raises(ValueError, match="no backward"):
        A.attention_prompt(q, k, k, cu, sinks=sinks)
    with pytest.raises(ValueError, match="no backward"):
        A.attention_shared(q, c[0].clone().requires_grad_(), c[0], c, c, n)
    with pytest.raises(ValueError, match="no backward"):
        A.cache_evict(c.clone().requires_grad_(), c, w, n, 4, 1)
    with pytest.raises(ValueError, match="no backward"):
        A.cache_evict(c, c, w.clone().requires_grad_(), n, 4, 1)
    before, out = w._version, torch.zeros_like(q)
    A.attention_shared(q, None, None, c, c, n, weights=w, out=out)
    assert w._version > before and out._version > 0
    before = out._version
    A.attention_prompt(q, k, k, cu, out=out)
    assert out._version > before
    with torch.inference_mode():
        A.attention_shared(q, None, None, c, c, n, weights=torch.zeros(4, 2, 8, device="cuda"), out=torch.zeros_like(q))


# ---- empty batches

def test_an_empty_batch_with_a_prefix_and_a_cache(A):
    bf = torch.bfloat16
    q, p, c = torch.ones(0, 32, 128, dtype=bf, device="cuda"), torch.ones(4, 16384, 128, dtype=bf, device="cuda"), \
        torch.ones(0, 4, 1024, 128, dtype=bf, device="cuda")
    n, w = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, 4, 1024, device="cuda")
    assert A.attention_shared(q, p, p, c, c, n, weights=w).shape == (0, 32, 128)


# ---- waits that run out

def test_a_wait_that_runs_out_is_reported_once(A, gpu):
    """The operators' waits end by themselves; tg_cuda_synchronize says so, and the next call is a good one."""
    assert gpu.tg_cuda_synchronize() == 0
    assert gpu.tg_cuda_debug_attn_wait() == 0
    assert gpu.tg_cuda_synchronize() == -1
    code, text = tg.last_error(gpu)
    assert code == 202 and "site 399 of an attention operator (3, 0)" in text, text
    assert gpu.tg_cuda_synchronize() == 0
    q, k = torch.ones(4, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert bool((A.attention_prompt(q, k, k, ends([4])) == 1).all())
    torch.cuda.synchronize()
    assert gpu.tg_cuda_synchronize() == 0
