"""Attention over device tensors for batched serving.

The layer steps of `layer.ResidentLayer` take batches of tokens that live on
the GPU; these operators are the attention between them, on torch CUDA
tensors of bfloat16 or float16:

  attention_prompt   causal attention of packed prompts (tg_attention_prompt)
  attention_shared   one token of each sequence over a shared prefix and its
                     own cache, gathering the keys' weights (tg_attention_shared)
  cache_evict        a cache cut to a budget by those weights (tg_cache_evict)

All are asynchronous on torch's current stream of the tensors' device, take
their workspace from torch's allocator, and can be captured in a CUDA graph.
Tensors may be strided views: the last dimension is contiguous, the other
strides are multiples of 8 elements, and data start on 16-byte boundaries.
head_dim is a multiple of 8, at most 128, and up to 128 query heads share a
key head.  Softmax statistics, accumulators and weights are fp32; the softmax
weights are rounded to the tensors' type for their product with the values.
What a query does not attend to (later positions, those before its window,
other sequences, rows behind a cache's lengths) may hold anything, infinities
and NaN too.  Bad arguments raise ValueError before anything runs
(ArgumentError, a TinyGiantCudaError too, where the library sees them); other
errors of the library raise TinyGiantCudaError.  There is no backward pass:
where autograd would record the call (gradients on, and a tensor that requires
them), it is refused.  Writes into out and weights count as changes in place.
"""
import ctypes

import torch

from . import TinyGiantCudaError, last_error, load

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_NO_TENSOR = (AttributeError, IndexError)          # of what is no tensor, or has no dimension
_I64x8, _I64x16 = ctypes.c_int64 * 8, ctypes.c_int64 * 16
_MOST = 0x7fffffff                                 # no position is beyond it
_empty = torch.empty_strided                       # less host time than torch.empty
_recording = torch.is_grad_enabled
_written = torch.autograd.graph.increment_version  # of tensors written in place
_raw_stream = torch._C._cuda_getCurrentRawStream   # torch.cuda.current_stream(i).cuda_stream, without its objects


class ArgumentError(TinyGiantCudaError, ValueError):
    """Arguments that the library refused."""


def _call(device, fn, *args):
    """One library call on torch's current stream of `device` (an index)."""
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(device, fn, *args)
    rc = fn(*args, _raw_stream(device))
    if rc:
        code, msg = last_error()
        raise (ArgumentError if rc == 3 else TinyGiantCudaError)(f"[{code}] {msg}")


def _window(n):
    """A window as the library's 32-bit argument: one beyond any position is as good as the largest."""
    if n < 0:
        raise ValueError(f"window must not be negative; is {n}")
    return n if n < _MOST else _MOST


def _ptr(t):
    return None if t is None else t.data_ptr()


# The calls below test their tensors in one expression each, since their whole
# host time is a few microseconds; _refuse says what is wrong when it fails.
# What the library can see (strides, counts, alignment) it tests itself.

def _refuse(named, heads=None, small=()):
    """Raises the ValueError of the first tensor that does not fit.  named: (name, tensor, dimensions, shape or None);
    heads: (H, KH, hd); small: (name, tensor, dtype, shape), None where a call may leave the tensor out."""
    def need(ok, text):
        if not ok:
            raise ValueError(text)

    _, first, _, _ = named[0]
    for name, t, ndim, shape in named:
        need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
        need(t.dim() == ndim, f"{name} must have {ndim} dimensions, has {t.dim()}")
        need(t.dtype in _DTYPES and t.dtype == first.dtype,
             f"{name} must be bfloat16 or float16, all of one type; is {t.dtype}")
        need(t.device == first.device, f"{name} must be on {first.device}, is on {t.device}")
        need(t.stride(-1) == 1, f"{name}'s last dimension must be contiguous")
    if heads:
        H, KH, hd = heads
        need(KH > 0 and H % KH == 0 and H // KH <= 128, f"{H} query heads do not share {KH} key heads (1 to 128 each)")
        need(0 < hd <= 128 and hd % 8 == 0, f"head_dim must be a multiple of 8, at most 128; is {hd}")
    for name, t, ndim, shape in named:
        need(shape is None or tuple(t.shape) == tuple(shape), f"{name} {tuple(t.shape)} and the others do not fit: must be {shape}")
    for name, t, dtype, shape in filter(None, small):
        need(isinstance(t, torch.Tensor) and t.device == first.device, f"{name} must be a tensor on {first.device}")
        need(t.dtype == dtype and tuple(t.shape) == tuple(shape), f"{name} must be {dtype} {tuple(shape)}, is {t.dtype} {tuple(t.shape)}")
        need(t.is_contiguous() or (name == "weights" and t.stride(2) == 1), f"{name} must be contiguous")
        need(name != "weights" or min(t.stride()) > 0, f"{name} must not be broadcast")
    raise ValueError("the tensors do not fit one another")


def _fits(t, device, dtype):
    return t.get_device() == device and t.dtype is dtype and t.stride()[-1] == 1


def _heads_of(q, k, dims):
    """dtype, device index, shape of q and (rows, heads, head_dim) of k, which has `dims` dimensions."""
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and q.dtype in _DTYPES and q.is_cuda and q.dim() == 3
            and k.dim() == dims):
        _refuse([("q", q, 3, None), ("k", k, dims, None)])
    H, KH, hd = q.shape[1], k.shape[1], q.shape[2]
    if KH == 0 or H % KH or H // KH > 128 or hd % 8 or not 0 < hd <= 128:
        _refuse([("q", q, 3, None)], (H, KH, hd))
    return q.dtype, q.get_device(), q.shape, (k.shape[0], KH, hd)


def _no_backward():
    if _recording():
        raise ValueError("the attention operators have no backward pass: call them under torch.no_grad(), or detach the tensors")


def _need_out(out, q):
    if not isinstance(out, torch.Tensor) or out.shape != q.shape:
        raise ValueError(f"out must have the shape of q, {tuple(q.shape)}")


def attention_prompt(q, k, v, cu_q, cu_k=None, *, max_k=None, window=0, sinks=None, scale=None, out=None):
    """Causal attention of sequences packed one after another.

    q [total_q, H, hd]; k, v [total_k, KH, hd], H a multiple of KH.  Sequence
    s has the rows cu_q[s] .. cu_q[s + 1] of q and cu_k[s] .. cu_k[s + 1] of k
    and v (int32 on the device, n + 1 ascending values from 0 to the total;
    cu_k None: cu_q).  Its queries are the last of its positions: with nq
    queries and nk keys, query i is at position nk - nq + i and attends to the
    keys up to it, the last `window` of them if window > 0.  sinks [H] fp32
    adds a logit without a value to each softmax.  scale: 1 / sqrt(hd).  A
    query without a key gives zeros.  max_k: the largest number of keys of a
    sequence, if known (default total_k); it sizes the workspace, and results
    depend on it by no more than the order of their fp32 sums (it decides how
    long axes are split).  A query whose scores have a NaN or +inf among its
    keys gives NaN, one whose scores are all -inf zeros.  Returns
    out [total_q, H, hd]; out must not overlap the inputs."""
    dtype, dev, (tq, H, hd), (tk, KH, _) = _heads_of(q, k, 3)
    n = cu_q.shape[0] - 1 if isinstance(cu_q, torch.Tensor) and cu_q.dim() == 1 else -1
    if cu_k is None:
        if tk != tq:
            raise ValueError(f"without cu_k there are as many keys as queries; got {tk} and {tq}")
        cu_k = cu_q
    given = out is not None
    if not given:
        out = _empty((tq, H, hd), (H * hd, hd, 1), dtype=dtype, device=q.device)
    try:
        fit = (dev >= 0 and n >= 0 and k.shape == v.shape and k.shape[2] == hd and out.shape == q.shape
               and _fits(q, dev, dtype) and _fits(k, dev, dtype) and _fits(v, dev, dtype) and _fits(out, dev, dtype)
               and _fits(cu_q, dev, torch.int32) and _fits(cu_k, dev, torch.int32) and cu_k.shape == cu_q.shape
               and (sinks is None or (_fits(sinks, dev, torch.float32) and sinks.shape == (H,))))
    except _NO_TENSOR:
        fit = False
    if not fit:
        _need_out(out, q)
        _refuse([("q", q, 3, None), ("k", k, 3, (tk, KH, hd)), ("v", v, 3, (tk, KH, hd)), ("out", out, 3, None)], (H, KH, hd),
                [("cu_q", cu_q, torch.int32, (max(n, 0) + 1,)), ("cu_k", cu_k, torch.int32, (max(n, 0) + 1,)),
                 sinks is not None and ("sinks", sinks, torch.float32, (H,))])
    if (q.requires_grad or k.requires_grad or v.requires_grad or (given and out.requires_grad)
            or (sinks is not None and sinks.requires_grad)):
        _no_backward()
    max_k = tk if max_k is None or max_k > tk else max_k
    lib = load()
    nbytes = lib.tg_attention_prompt_workspace(n, tq, max_k, H, KH, hd)
    ws = _empty((nbytes,), (1,), dtype=torch.uint8, device=q.device) if nbytes else None
    (q0, q1, _), (k0, k1, _), (v0, v1, _), (o0, o1, _) = q.stride(), k.stride(), v.stride(), out.stride()
    _call(dev, lib.tg_attention_prompt, _DTYPES[dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
          cu_q.data_ptr(), cu_k.data_ptr(), _ptr(sinks), n, tq, tk, max_k, H, KH, hd,
          _I64x8(q0, q1, k0, k1, v0, v1, o0, o1), _window(window), hd ** -0.5 if scale is None else scale, _ptr(ws), nbytes)
    if given:
        _written(out)
    return out


def attention_shared(q, prefix_k, prefix_v, k, v, lens, *, max_len=None, window=0, sinks=None, scale=None, weights=None,
                     out=None):
    """One new token of each sequence over a shared prefix and its own cache.

    q [B, H, hd]; prefix_k, prefix_v [KH, P, hd] (None: no prefix), read once
    for every 256 query rows of a key head (32 sequences of 8 heads); k, v
    [B, KH, cap, hd], read once for every 16 query heads of a key head; lens
    [B] int32 on the device: the own positions of each sequence, its newest
    token's key the last of them.  The prefix is at the positions 0 .. P - 1,
    the own keys behind it.  window > 0: only the last `window` positions, as
    rows of the cache count them: after cache_evict has closed the gaps that is
    not the last `window` tokens.  sinks, scale: as attention_prompt.  weights
    [B, KH, cap] fp32: each own key's softmax weight, summed over the query heads that share it, is added in place.
    max_len: an upper bound of lens (default cap); a larger value in lens
    counts as max_len.  A sequence without a key gives zeros.  Rows of the
    caches behind lens are not read as values: they may hold anything.
    Returns out [B, H, hd]."""
    dtype, dev, (B, H, hd), (_, KH, _) = _heads_of(q, k, 4)
    P = 0 if prefix_k is None else prefix_k.shape[1] if isinstance(prefix_k, torch.Tensor) and prefix_k.dim() == 3 else -1
    given = out is not None
    if not given:
        out = _empty((B, H, hd), (H * hd, hd, 1), dtype=dtype, device=q.device)
    try:
        fit = (dev >= 0 and k.shape == v.shape and k.shape[0] == B and k.shape[3] == hd and out.shape == q.shape
               and _fits(q, dev, dtype) and _fits(k, dev, dtype) and _fits(v, dev, dtype) and _fits(out, dev, dtype)
               and (prefix_k is None if prefix_v is None else
                    prefix_k is not None and prefix_k.shape == prefix_v.shape == (KH, P, hd) and _fits(prefix_k, dev, dtype)
                    and _fits(prefix_v, dev, dtype))
               and _fits(lens, dev, torch.int32) and lens.shape == (B,)
               and (sinks is None or (_fits(sinks, dev, torch.float32) and sinks.shape == (H,)))
               and (weights is None or (_fits(weights, dev, torch.float32) and weights.shape == k.shape[:3]
                                        and min(weights.stride()) > 0)))
    except _NO_TENSOR:
        fit = False
    if not fit:
        _need_out(out, q)
        cap = k.shape[2]
        named = [("q", q, 3, None), ("k", k, 4, (B, KH, cap, hd)), ("v", v, 4, (B, KH, cap, hd)), ("out", out, 3, None)]
        if prefix_k is not None or prefix_v is not None:
            if not all(isinstance(t, torch.Tensor) and t.shape == (KH, P, hd) for t in (prefix_k, prefix_v)):
                raise ValueError(f"prefix_k and prefix_v must both be [{KH}, P, {hd}]")
            named += [("prefix_k", prefix_k, 3, None), ("prefix_v", prefix_v, 3, None)]
        _refuse(named, (H, KH, hd), [("lens", lens, torch.int32, (B,)), sinks is not None and ("sinks", sinks, torch.float32, (H,)),
                                     weights is not None and ("weights", weights, torch.float32, (B, KH, cap))])
    if (q.requires_grad or k.requires_grad or v.requires_grad or (given and out.requires_grad)
            or (P and (prefix_k.requires_grad or prefix_v.requires_grad)) or (sinks is not None and sinks.requires_grad)
            or (weights is not None and weights.requires_grad)):
        _no_backward()
    cap = k.shape[2]
    max_len = cap if max_len is None or max_len > cap else max_len
    lib = load()
    nbytes = lib.tg_attention_shared_workspace(B, P, max_len, H, KH, hd, weights is not None)
    ws = _empty((nbytes,), (1,), dtype=torch.uint8, device=q.device) if nbytes else None
    (q0, q1, _), (o0, o1, _), (k0, k1, k2, _), (v0, v1, v2, _) = q.stride(), out.stride(), k.stride(), v.stride()
    (pk0, pk1, _), (pv0, pv1, _) = (prefix_k.stride(), prefix_v.stride()) if P else ((8, 8, 1), (8, 8, 1))
    w0, w1, _ = weights.stride() if weights is not None else (1, 1, 1)
    _call(dev, lib.tg_attention_shared, _DTYPES[dtype], q.data_ptr(), _ptr(prefix_k), _ptr(prefix_v), k.data_ptr(),
          v.data_ptr(), out.data_ptr(), lens.data_ptr(), _ptr(sinks), _ptr(weights), B, P, cap, max_len, H, KH, hd,
          _I64x16(q0, q1, pk0, pk1, pv0, pv1, k0, k1, k2, v0, v1, v2, o0, o1, w0, w1), _window(window),
          hd ** -0.5 if scale is None else scale, _ptr(ws), nbytes)
    if given:
        _written(out)
    if weights is not None:
        _written(weights)
    return out


def cache_evict(k, v, weights, lens, keep, recent):
    """A cache cut down to `keep` positions of each sequence and key head.

    k, v [B, KH, cap, hd]; weights [B, KH, cap] fp32, as attention_shared
    gathers them; lens [B] int32 on the device.  Of a sequence's n positions
    min(n, keep) stay: the last `recent` of them, and of the others those of
    the largest weight (equal weights: the earlier position; NaN counts as the
    largest).  Weights come from decoded tokens: straight after a prompt they
    are all zero, and the earliest positions stay.  Each key head keeps its own
    choice, in the order they had; rows are moved together, so windows of later
    calls count kept rows, not tokens.  B x KH is at most 65535.
    Returns (k, v, weights, lens, indices): new tensors [B, KH, keep, hd],
    [B, KH, keep, hd], [B, KH, keep], [B] and the positions' old places
    [B, KH, keep] int32; behind a sequence's end they hold zeros and -1."""
    try:
        shape, dtype, dev = k.shape, k.dtype, k.get_device()
        fit = (len(shape) == 4 and dtype in _DTYPES and dev >= 0 and shape == v.shape and weights.shape == shape[:3]
               and _fits(k, dev, dtype) and _fits(v, dev, dtype) and _fits(weights, dev, torch.float32)
               and min(weights.stride()) > 0 and _fits(lens, dev, torch.int32) and lens.shape == shape[:1])
    except _NO_TENSOR:
        fit = False
    if not fit:
        tensors = isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)
        if tensors and k.shape != v.shape:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape")
        _refuse([("k", k, 4, None), ("v", v, 4, None)], None,
                [("weights", weights, torch.float32, k.shape[:3]), ("lens", lens, torch.int32, k.shape[:1])] if tensors else ())
    if k.requires_grad or v.requires_grad or weights.requires_grad:
        _no_backward()
    B, KH, cap, hd = shape
    where = k.device
    if not (0 < keep <= cap and 0 <= recent <= keep):
        raise ValueError(f"need 0 < keep <= {cap} and 0 <= recent <= keep; got {keep}, {recent}")
    rows = KH * keep
    ko = _empty((B, KH, keep, hd), (rows * hd, keep * hd, hd, 1), dtype=dtype, device=where)
    vo = torch.empty_like(ko)
    wo = _empty((B, KH, keep), (rows, keep, 1), dtype=torch.float32, device=where)
    idx = _empty((B, KH, keep), (rows, keep, 1), dtype=torch.int32, device=where)
    lo = _empty((B,), (1,), dtype=torch.int32, device=where)
    (k0, k1, k2, _), (v0, v1, v2, _), (w0, w1, _) = k.stride(), v.stride(), weights.stride()
    _call(dev, load().tg_cache_evict, k.data_ptr(), v.data_ptr(), weights.data_ptr(), lens.data_ptr(), ko.data_ptr(),
          vo.data_ptr(), wo.data_ptr(), lo.data_ptr(), idx.data_ptr(), B, cap, KH, hd,
          _I64x8(k0, k1, k2, v0, v1, v2, w0, w1), keep, recent)
    return ko, vo, wo, lo, idx
