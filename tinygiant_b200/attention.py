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
head_dim is a multiple of 8, at most 128.  Softmax statistics, accumulators
and weights are fp32.  Bad arguments raise ValueError before anything runs;
an error of the library raises TinyGiantCudaError.
"""
import ctypes
import math

import torch

from . import TinyGiantCudaError, last_error, load

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _data(t, name, ndim, like=None):
    """Checks a 16-bit tensor; its strides, with 8 in the place of those that no index uses."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
    _need(t.dim() == ndim, f"{name} must have {ndim} dimensions, has {t.dim()}")
    _need(t.dtype in _DTYPES if like is None else t.dtype == like.dtype,
          f"{name} must be bfloat16 or float16, all of one type; is {t.dtype}")
    _need(like is None or t.device == like.device, f"{name} must be on {like.device if like is not None else ''}")
    shape, st = t.shape, t.stride()
    _need(st[-1] == 1 or shape[-1] == 1, f"{name}'s last dimension must be contiguous")
    out = []
    for n, s in zip(shape[:-1], st[:-1]):
        if n <= 1:
            s = 8
        elif s <= 0 or s % 8:
            raise ValueError(f"{name}'s strides must be positive multiples of 8 elements, are {tuple(st)}")
        out.append(s)
    return out


def _small(t, name, dtype, shape, like):
    _need(isinstance(t, torch.Tensor) and t.device == like.device, f"{name} must be a tensor on {like.device}")
    _need(t.dtype == dtype and tuple(t.shape) == tuple(shape) and t.is_contiguous(),
          f"{name} must be contiguous {dtype} of shape {tuple(shape)}, is {t.dtype} {tuple(t.shape)}")


def _heads(H, KH, hd):
    _need(KH > 0 and H % KH == 0 and H // KH <= 128, f"{H} query heads do not share {KH} key heads (1 to 128 each)")
    _need(0 < hd <= 128 and hd % 8 == 0, f"head_dim must be a multiple of 8, at most 128; is {hd}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(device, fn, *args):
    """One library call on torch's current stream of `device`."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(device, fn, *args)
    if fn(*args, torch.cuda.current_stream(device).cuda_stream):
        code, msg = last_error()
        raise TinyGiantCudaError(f"[{code}] {msg}")


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
    do not depend on it.  Returns out [total_q, H, hd]; out must not overlap
    the inputs."""
    sq, sk, sv = _data(q, "q", 3), _data(k, "k", 3, q), _data(v, "v", 3, q)
    (tq, H, hd), (tk, KH, _) = q.shape, k.shape
    _heads(H, KH, hd)
    _need(k.shape == v.shape and k.shape[2] == hd, f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    _need(isinstance(cu_q, torch.Tensor) and cu_q.dim() == 1 and len(cu_q) >= 1, "cu_q must have one value more than there are sequences")
    _small(cu_q, "cu_q", torch.int32, cu_q.shape, q)
    if cu_k is None:
        _need(tk == tq, "without cu_k there are as many keys as queries")
        cu_k = cu_q
    else:
        _small(cu_k, "cu_k", torch.int32, cu_q.shape, q)
    if sinks is not None:
        _small(sinks, "sinks", torch.float32, (H,), q)
    _need(window >= 0, "window must not be negative")
    max_k = tk if max_k is None else min(max_k, tk)
    _need(max_k >= 0, "max_k must not be negative")
    if out is None:
        out = torch.empty(tq, H, hd, dtype=q.dtype, device=q.device)
    so = _data(out, "out", 3, q)
    _need(out.shape == q.shape, f"out must have the shape of q, {tuple(q.shape)}")
    if tq == 0:
        return out
    lib, n = load(), len(cu_q) - 1
    nbytes = lib.tg_attention_prompt_workspace(n, tq, max_k, H, KH, hd)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _call(q.device, lib.tg_attention_prompt, _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
          cu_q.data_ptr(), cu_k.data_ptr(), _ptr(sinks), n, tq, tk, max_k, H, KH, hd,
          (ctypes.c_int64 * 8)(*sq, *sk, *sv, *so), window, 1.0 / math.sqrt(hd) if scale is None else scale, _ptr(ws),
          nbytes)
    return out


def attention_shared(q, prefix_k, prefix_v, k, v, lens, *, max_len=None, window=0, sinks=None, scale=None, weights=None,
                     out=None):
    """One new token of each sequence over a shared prefix and its own cache.

    q [B, H, hd]; prefix_k, prefix_v [KH, P, hd] (None: no prefix), read once
    for the whole batch; k, v [B, KH, cap, hd]; lens [B] int32 on the device:
    the own positions of each sequence, its newest token's key the last of
    them.  The prefix is at the positions 0 .. P - 1, the own keys behind it.
    window > 0: only the last `window` positions.  sinks, scale: as
    attention_prompt.  weights [B, KH, cap] fp32: each own key's softmax
    weight, summed over the query heads that share it, is added in place.
    max_len: an upper bound of lens (default cap); a larger value in lens
    counts as max_len.  A sequence without a key gives zeros.  Rows of the
    caches behind lens are not read as values: they may hold anything.
    Returns out [B, H, hd]."""
    sq, sk, sv = _data(q, "q", 3), _data(k, "k", 4, q), _data(v, "v", 4, q)
    (B, H, hd), (_, KH, cap, _) = q.shape, k.shape
    _heads(H, KH, hd)
    _need(k.shape == v.shape and tuple(k.shape) == (B, KH, cap, hd),
          f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    P, sp = 0, [8, 8, 8, 8]
    if prefix_k is not None:
        sp = _data(prefix_k, "prefix_k", 3, q)
        P = prefix_k.shape[1]
        _need(prefix_v is not None and prefix_k.shape == prefix_v.shape and tuple(prefix_k.shape) == (KH, P, hd),
              f"prefix_k and prefix_v must both be [{KH}, P, {hd}]")
        sp = sp + _data(prefix_v, "prefix_v", 3, q)
    _small(lens, "lens", torch.int32, (B,), q)
    if sinks is not None:
        _small(sinks, "sinks", torch.float32, (H,), q)
    sw = (1, 1)
    if weights is not None:
        _need(isinstance(weights, torch.Tensor) and weights.device == q.device and weights.dtype == torch.float32
              and tuple(weights.shape) == (B, KH, cap) and (cap <= 1 or weights.stride(2) == 1),
              f"weights must be float32 [{B}, {KH}, {cap}] with contiguous rows")
        sw = [s if n > 1 else 1 for n, s in zip(weights.shape[:2], weights.stride()[:2])]
        _need(min(sw) > 0, "weights must not be broadcast")
    _need(window >= 0, "window must not be negative")
    max_len = cap if max_len is None else min(max_len, cap)
    _need(max_len >= 0, "max_len must not be negative")
    if out is None:
        out = torch.empty(B, H, hd, dtype=q.dtype, device=q.device)
    so = _data(out, "out", 3, q)
    _need(out.shape == q.shape, f"out must have the shape of q, {tuple(q.shape)}")
    if B == 0:
        return out
    lib = load()
    nbytes = lib.tg_attention_shared_workspace(B, P, max_len, H, KH, hd, weights is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _call(q.device, lib.tg_attention_shared, _DTYPES[q.dtype], q.data_ptr(), _ptr(prefix_k), _ptr(prefix_v), k.data_ptr(),
          v.data_ptr(), out.data_ptr(), lens.data_ptr(), _ptr(sinks), _ptr(weights), B, P, cap, max_len, H, KH, hd,
          (ctypes.c_int64 * 16)(*sq, *sp, *sk, *sv, *so, *sw), window, 1.0 / math.sqrt(hd) if scale is None else scale,
          _ptr(ws), nbytes)
    return out


def cache_evict(k, v, weights, lens, keep, recent):
    """A cache cut down to `keep` positions of each sequence and key head.

    k, v [B, KH, cap, hd]; weights [B, KH, cap] fp32, as attention_shared
    gathers them; lens [B] int32 on the device.  Of a sequence's n positions
    min(n, keep) stay: the last `recent` of them, and of the others those of
    the largest weight (equal weights: the earlier position; NaN counts as the
    largest).  Each key head keeps its own choice, in the order they had.
    Returns (k, v, weights, lens, indices): new tensors [B, KH, keep, hd],
    [B, KH, keep, hd], [B, KH, keep], [B] and the positions' old places
    [B, KH, keep] int32; behind a sequence's end they hold zeros and -1."""
    sk, sv = _data(k, "k", 4), _data(v, "v", 4, k)
    B, KH, cap, hd = k.shape
    _heads(KH, KH, hd)
    _need(k.shape == v.shape, f"k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape")
    _need(isinstance(weights, torch.Tensor) and weights.device == k.device and weights.dtype == torch.float32
          and tuple(weights.shape) == (B, KH, cap) and (cap <= 1 or weights.stride(2) == 1),
          f"weights must be float32 [{B}, {KH}, {cap}] with contiguous rows")
    sw = [s if n > 1 else 1 for n, s in zip(weights.shape[:2], weights.stride()[:2])]
    _need(min(sw) > 0, "weights must not be broadcast")
    _small(lens, "lens", torch.int32, (B,), k)
    _need(0 < keep <= cap and 0 <= recent <= keep, f"need 0 < keep <= {cap} and 0 <= recent <= keep; got {keep}, {recent}")
    ko, vo = (torch.empty(B, KH, keep, hd, dtype=k.dtype, device=k.device) for _ in range(2))
    wo = torch.empty(B, KH, keep, dtype=torch.float32, device=k.device)
    idx = torch.empty(B, KH, keep, dtype=torch.int32, device=k.device)
    lo = torch.empty(B, dtype=torch.int32, device=k.device)
    if B:
        _call(k.device, load().tg_cache_evict, k.data_ptr(), v.data_ptr(), weights.data_ptr(), lens.data_ptr(),
              ko.data_ptr(), vo.data_ptr(), wo.data_ptr(), lo.data_ptr(), idx.data_ptr(), B, cap, KH, hd,
              (ctypes.c_int64 * 8)(*sk, *sv, *sw), keep, recent)
    return ko, vo, wo, lo, idx
