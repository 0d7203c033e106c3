"""A paged key/value cache on device tensors, and positions: what a server of
batched steps has between its layer steps when sequences come and go.

  rotary_frequencies   angles per position, scaled for long contexts
  rotary               queries and keys rotated by their positions (tg_rotary)
  cache_append         new tokens' keys and values into their pages, rotated
                       on the way (tg_paged_append)
  attention_paged      the newest tokens of each sequence over its pages
                       (tg_attention_paged)
  cache_gather         pages read back as packed keys and values, for
                       attention.attention_prompt (tg_paged_gather)

A cache is two pools of pages, k_pages and v_pages [n_pages, KH, page, hd], and
a table of page numbers for each sequence, tables [B, columns] int32: position
p of sequence b is row p % page of the page tables[b, p // page].  page is a
power of two, at least 16.  Numbers outside the pool (-1, say) are no pages:
what would lie there is not written, has no weight, and reads as zeros, so
pages behind a window can be given back.  Sequences may share pages that
neither writes.

Pages are of the tensors' own type, bfloat16 or float16, or of 8 bits,
torch.float8_e4m3fn with scales k_scales and v_scales [n_pages, KH, page // 16]
fp32: a value is its code times the scale of its block of 16 positions and key
head.  cache_append makes scales that are powers of two, the least (but 2^-117
at least) under which a block's values reach no further than 448; a larger
token raises its block's scale, and the codes before it in the block are
rounded again.  A first token of a block starts its scale anew, whatever was
there.  attention_paged and cache_gather take any positive scales, and
cache_append keeps one that it finds before a block's new tokens where it is
the larger.

As in tinygiant_b200.attention: calls are asynchronous on torch's current
stream of the tensors' device, take workspace and outputs from torch's
allocator, can be captured in a CUDA graph, give the same bits each time, and
read lengths and tables on the device.  Tensors may be strided views: the last
dimension is contiguous, the other strides are multiples of 16 bytes (scales
and tables: any, all dimensions of scales), none is broadcast, and data start
on 16-byte boundaries.  head_dim is a
multiple of 8 (16 for pages of 8 bits), at most 128.  Norms, angles, rotations,
softmax statistics and accumulators are fp32 or more.  Bad arguments raise
ValueError before anything runs; there is no backward pass.
"""
import ctypes
import math
import struct

import torch

from . import TinyGiantCudaError, last_error, load
from .attention import _DTYPES, _MOST, ArgumentError, _empty, _forward, _no_backward, _no_tangents, _raw_stream, _window, _written

__all__ = ["rotary_frequencies", "rotary", "cache_append", "attention_paged", "cache_gather", "ArgumentError"]

_CODES = torch.float8_e4m3fn
_F32, _F64, _I32 = torch.float32, torch.float64, torch.int32
_current = torch._C._cuda_getDevice
_MISFITS = (AttributeError, IndexError, KeyError, TypeError, ValueError)   # of what is no tensor, or of other dimensions
# The calls' arguments as tg_paged_call's records: a call of 30 arguments through ctypes takes 7 us, a record of them 1.
_ROTARY, _APPEND, _ATTEND, _GATHER = (struct.Struct(f).pack for f in ("24q2dq", "49q2dq", "41qd3q", "36q"))


def _run(device, record):
    """One library call on the tensors' device (an index)."""
    if device != _current():
        with torch.cuda.device(device):
            rc = load().tg_paged_call(record)
    else:
        rc = load().tg_paged_call(record)
    if rc:
        code, msg = last_error()
        raise (ArgumentError if rc == 3 else TinyGiantCudaError)(f"[{code}] {msg}")


def _no_number(e):
    """What struct cannot pack or ctypes pass: a number that is none, or beyond 64 bits."""
    raise ValueError(f"bad argument: {e}") from None


def rotary_frequencies(dim, theta=10000.0, *, scaling=None, factor=1.0, original_len=None, beta_fast=32.0, beta_slow=1.0,
                       truncate=True, device=None):
    """The angles per position of `dim` rotated dimensions, and the amplitude.

    Pair j of dim // 2 turns by theta^(-2 j / dim) radians a position.  scaling,
    for contexts `factor` times as long: "linear" divides all by factor; "ntk"
    raises theta by factor^(dim / (dim - 2)); "yarn" divides those that turn
    less than beta_slow times in original_len positions, leaves those that turn
    more than beta_fast times, goes evenly over the pairs between (whose ends
    are whole pairs if truncate), and has the amplitude 0.1 ln(factor) + 1.
    Returns (fp64 tensor [dim // 2], float)."""
    if dim <= 0 or dim % 2 or not theta > 1 or not factor >= 1:
        raise ValueError(f"need an even dim > 0, theta > 1 and factor >= 1; got {dim}, {theta}, {factor}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn'; is {scaling!r}")
    if scaling == "ntk":
        if dim <= 2:
            raise ValueError("'ntk' needs more than one pair")
        theta = theta * factor ** (dim / (dim - 2))
    f = [theta ** (-2 * j / dim) for j in range(dim // 2)]
    amplitude = 1.0
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":
        if not original_len or original_len < 1 or not beta_fast >= beta_slow > 0:
            raise ValueError("'yarn' needs original_len >= 1 and beta_fast >= beta_slow > 0")
        low, high = (dim * math.log(original_len / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (beta_fast, beta_slow))
        if truncate:
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, dim - 1)
        less = [min(1.0, max(0.0, (j - low) / max(high - low, 0.001))) for j in range(dim // 2)]
        f = [x / factor * w + x * (1 - w) for x, w in zip(f, less)]
        amplitude = 0.1 * math.log(factor) + 1
    return torch.tensor(f, dtype=torch.float64, device=device), amplitude


# As in tinygiant_b200.attention, each call tests its tensors in one
# expression, and _refuse says what is wrong when that fails.

def _refuse(first, *named):
    """Raises the ValueError of the first tensor that does not fit.  named: (name, tensor, dtypes, shape), a shape's -1 for any
    number, None for what a call may leave out; first: the tensor that the others go by."""
    for name, t, dtypes, shape in filter(None, named):
        if not (isinstance(t, torch.Tensor) and t.is_cuda):
            raise ValueError(f"{name} must be a CUDA tensor")
        if t.device != first.device:
            raise ValueError(f"{name} must be on {first.device}, is on {t.device}")
        if t.dtype not in dtypes:
            raise ValueError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}; is {t.dtype}")
        if t.dim() != len(shape) or any(n not in (-1, m) for n, m in zip(shape, t.shape)):
            raise ValueError(f"{name} {tuple(t.shape)} and the others do not fit: must be {tuple(shape)}")
        if t.stride(-1) != 1 and not name.endswith("scales"):
            raise ValueError(f"{name}'s last dimension must be contiguous")
    raise ValueError("the tensors do not fit one another")


def _vector(t, dev, dtype, n):
    """Whether t is a contiguous vector of n values."""
    return t.dtype is dtype and t.get_device() == dev and t.shape == (n,) and (n < 2 or t.stride() == (1,))


def _pool(dev, dtype, k_pages, v_pages, tables, k_scales, v_scales, KH, hd):
    """The cache's strides as the library takes them, or None where pools, scales and tables do not fit key heads of `dtype`;
    AttributeError, IndexError or ValueError for what is no tensor, or of other dimensions."""
    shape, kind = k_pages.shape, k_pages.dtype
    N, kh, page, d = shape
    k0, k1, k2, k3 = k_pages.stride()
    v0, v1, v2, v3 = v_pages.stride()
    t0, t1 = tables.stride()
    if not (kh == KH and d == hd and v_pages.shape == shape and v_pages.dtype is kind and k3 == v3 == t1 == 1
            and tables.dtype is _I32 and k_pages.get_device() == v_pages.get_device() == tables.get_device() == dev):
        return None
    if kind is _CODES:
        if not (k_scales.shape == v_scales.shape == (N, kh, page // 16) and k_scales.dtype is v_scales.dtype is _F32
                and k_scales.get_device() == v_scales.get_device() == dev):
            return None
        return (k0, k1, k2, v0, v1, v2, *k_scales.stride(), *v_scales.stride(), t0)
    if kind is not dtype or k_scales is not None or v_scales is not None:
        return None
    return (k0, k1, k2, v0, v1, v2, 1, 1, 1, 1, 1, 1, t0)


def _pool_named(dtype, k_pages, v_pages, tables, k_scales, v_scales, B, KH, hd):
    """The same for _refuse; what it cannot say is raised here."""
    kinds = (dtype, _CODES)
    shape = tuple(k_pages.shape) if isinstance(k_pages, torch.Tensor) and k_pages.dim() == 4 else (-1, -1, -1, -1)
    codes = isinstance(k_pages, torch.Tensor) and k_pages.dtype is _CODES
    if not codes and (k_scales is not None or v_scales is not None):
        raise ValueError("pages of 16 bits have no scales")
    if codes and (k_scales is None or v_scales is None):
        raise ValueError("pages of 8 bits need k_scales and v_scales")
    return [("k_pages", k_pages, kinds, (shape[0], KH, shape[2], hd)),
            ("v_pages", v_pages, (k_pages.dtype,) if isinstance(k_pages, torch.Tensor) else kinds, shape),
            codes and ("k_scales", k_scales, (torch.float32,), (shape[0], KH, shape[2] // 16)),
            codes and ("v_scales", v_scales, (torch.float32,), (shape[0], KH, shape[2] // 16)),
            ("tables", tables, (torch.int32,), (B, -1))]


def rotary(q, k, positions, freqs, *, interleaved=False, amplitude=1.0, q_norm=None, k_norm=None, eps=1e-6, out=None):
    """Queries and keys rotated by their tokens' positions.

    q [T, H, hd] and k [T, KH, hd] (or None); positions [T] int32; freqs [n]
    fp64, the angles per position in radians (rotary_frequencies), 2 n <= hd.
    Pair j of a head is its dimensions (j, j + n), or (2 j, 2 j + 1) if
    interleaved; dimensions from 2 n on stay as they are.  The pairs are
    multiplied by amplitude.  q_norm, k_norm [hd] fp32: each head is first
    divided by sqrt(mean(x^2) + eps) and multiplied by these; the squares are
    summed in fp32, so heads of 2^64 are normed to zero, and with an eps of
    nothing heads below 2^-60 lose bits.
    out: (q, k) to write, which may be q and k themselves but must not overlap
    them in any other way.  Returns (q, k), k None if it was."""
    given = out is not None
    try:
        dtype, dev, (T, H, hd), (q0, q1, q2) = q.dtype, q.get_device(), q.shape, q.stride()
        kind = _DTYPES[dtype]
        if given:
            qo, ko = out
            o0, o1, o2 = qo.stride()
            fit = qo.dtype is dtype and qo.get_device() == dev and qo.shape == q.shape
        else:
            o0, o1, o2 = max(H, 1) * hd, hd, 1
            qo, ko, fit = _empty((T, H, hd), (o0, o1, 1), dtype=dtype, device=q.device), None, True
        if k is None:
            KH, k0, k1, k2, p0, p1, p2, fit = 0, 8, 8, 1, 8, 8, 1, fit and ko is None
        else:
            (k0, k1, k2), KH = k.stride(), k.shape[1]
            if given:
                p0, p1, p2 = ko.stride()
                fit = fit and ko.dtype is dtype and ko.get_device() == dev and ko.shape == k.shape
            else:
                p0, p1, p2 = max(KH, 1) * hd, hd, 1
                ko = _empty((T, KH, hd), (p0, p1, 1), dtype=dtype, device=q.device)
            fit = fit and k.dtype is dtype and k.get_device() == dev and k.shape == (T, KH, hd)
        n, = freqs.shape
        fit = (fit and dev >= 0 and q2 == k2 == o2 == p2 == 1 and positions is not None and _vector(positions, dev, _I32, T)
               and _vector(freqs, dev, _F64, n) and (q_norm is None or _vector(q_norm, dev, _F32, hd))
               and (k_norm is None or _vector(k_norm, dev, _F32, hd)))
    except _MISFITS:
        fit = False
    if not fit:
        _refuse_rotary(q, k, positions, freqs, q_norm, k_norm, out)
    if (q.requires_grad or (k is not None and (k.requires_grad or ko.requires_grad)) or freqs.requires_grad or qo.requires_grad
            or (q_norm is not None and q_norm.requires_grad) or (k_norm is not None and k_norm.requires_grad)):
        _no_backward()
    if _forward._current_level >= 0:
        _no_tangents(q, k, freqs, q_norm, k_norm, qo, ko)
    try:
        record = _ROTARY(0, kind, q.data_ptr(), 0 if k is None else k.data_ptr(), qo.data_ptr(), 0 if k is None else ko.data_ptr(),
                         positions.data_ptr(), freqs.data_ptr(), 0 if q_norm is None else q_norm.data_ptr(),
                         0 if k_norm is None else k_norm.data_ptr(), T, H, KH, hd, n, interleaved, q0, q1, k0, k1, o0, o1, p0, p1,
                         amplitude, eps, _raw_stream(dev))
    except (struct.error, OverflowError) as e:
        _no_number(e)
    _run(dev, record)
    if given:
        _written(qo)
        if ko is not None:
            _written(ko)
    return qo, ko


def _refuse_rotary(q, k, positions, freqs, q_norm, k_norm, out):
    kinds, f32 = tuple(_DTYPES), (torch.float32,)
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype not in kinds:
        _refuse(q, ("q", q, kinds, (-1, -1, -1)))
    T, H, hd = q.shape
    same = (q.dtype,)
    qo, ko = (None, None) if out is None else out if isinstance(out, (tuple, list)) and len(out) == 2 else (out, out)
    _refuse(q, ("q", q, kinds, (T, H, hd)), k is not None and ("k", k, same, (T, -1, hd)),
            ("positions", positions, (torch.int32,), (T,)), ("freqs", freqs, (torch.float64,), (-1,)),
            q_norm is not None and ("q_norm", q_norm, f32, (hd,)), k_norm is not None and ("k_norm", k_norm, f32, (hd,)),
            out is not None and ("out[0]", qo, same, (T, H, hd)),
            out is not None and (k is not None or ko is not None) and ("out[1]", ko, same, tuple(k.shape) if k is not None else (0,)))


def cache_append(k, v, k_pages, v_pages, tables, lens, cu=None, *, k_scales=None, v_scales=None, freqs=None, positions=None,
                 interleaved=False, amplitude=1.0, q=None, q_norm=None, k_norm=None, eps=1e-6, out=None):
    """New tokens' keys, rotated on the way, and values written to their pages.

    k, v [T, KH, hd]: the new tokens of all sequences packed one after another,
    sequence b's the rows cu[b] .. cu[b + 1] (int32 on the device, B + 1
    ascending values; None: T / B of each).  lens [B] int32: the positions of
    each sequence with its new tokens, which are its last.  freqs, interleaved,
    amplitude, q_norm, k_norm and eps: as rotary; without freqs nothing is
    rotated.  positions [T] int32: what to rotate by, if it is not the place in
    the cache.  q [T, H, hd]: rotated as well and returned, in out if given
    (which may be q itself).  A token whose place is no place (a position below
    zero or behind the table, a page outside the pool) is not written there;
    its query is rotated all the same.  Rows of no sequence are left out, the
    query's too.  No place may be written twice in a call, and in pages of 8
    bits no two sequences may write to one block: its values would be undefined.
    In 8 bits scales and codes are those of the formulas in 64 bits, whatever
    order fp32 would have summed in (rotary's limits of a head's squares hold
    here too); a value that is not finite in fp32 becomes NaN and does not count
    for the scale.  Returns the rotated q, or None."""
    given = out is not None
    try:
        dtype, dev, shape, (k0, k1, k2), (v0, v1, v2) = k.dtype, k.get_device(), k.shape, k.stride(), v.stride()
        kind, (T, KH, hd) = _DTYPES[dtype], shape
        B, = lens.shape
        pool = _pool(dev, dtype, k_pages, v_pages, tables, k_scales, v_scales, KH, hd)
        N, _, page, _ = k_pages.shape
        rows, cols = tables.shape
        fit = (pool and dev >= 0 and k2 == v2 == 1 and v.shape == shape and v.dtype is dtype and v.get_device() == dev and rows == B
               and _vector(lens, dev, _I32, B)
               and ((T % B == 0 if B else T == 0) if cu is None else _vector(cu, dev, _I32, B + 1)))
        if q is None:
            H, q0, q1, o0, o1, fit = 0, 8, 8, 8, 8, fit and out is None
        else:
            (q0, q1, q2), H = q.stride(), q.shape[1]
            if given:
                o0, o1, o2 = out.stride()
                fit = fit and o2 == 1 and out.dtype is dtype and out.get_device() == dev and out.shape == q.shape
            else:
                o0, o1 = max(H, 1) * hd, hd
                out = _empty((T, H, hd), (o0, o1, 1), dtype=dtype, device=k.device)
            fit = fit and q2 == 1 and q.dtype is dtype and q.get_device() == dev and q.shape == (T, H, hd)
        n = 0
        if freqs is not None:
            n, = freqs.shape
            fit = fit and _vector(freqs, dev, _F64, n)
        fit = (fit and (positions is None or _vector(positions, dev, _I32, T))
               and (q_norm is None or _vector(q_norm, dev, _F32, hd)) and (k_norm is None or _vector(k_norm, dev, _F32, hd)))
    except _MISFITS:
        fit = False
    if not fit:
        _refuse_append(k, v, k_pages, v_pages, tables, lens, cu, k_scales, v_scales, freqs, positions, q, q_norm, k_norm,
                       out if given else None)
    if (k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad
            or (k_scales is not None and (k_scales.requires_grad or v_scales.requires_grad)) or (freqs is not None and freqs.requires_grad)
            or (q is not None and (q.requires_grad or out.requires_grad)) or (q_norm is not None and q_norm.requires_grad)
            or (k_norm is not None and k_norm.requires_grad)):
        _no_backward()
    if _forward._current_level >= 0:
        _no_tangents(k, v, k_pages, v_pages, k_scales, v_scales, freqs, q, q_norm, k_norm, out)
    try:
        record = _APPEND(1, kind, 16 if k_scales is None else 8, 0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(),
                         0 if q is None else out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                         0 if k_scales is None else k_scales.data_ptr(), 0 if k_scales is None else v_scales.data_ptr(), tables.data_ptr(),
                         lens.data_ptr(), 0 if cu is None else cu.data_ptr(), 0 if positions is None else positions.data_ptr(),
                         0 if freqs is None else freqs.data_ptr(), 0 if q_norm is None else q_norm.data_ptr(),
                         0 if k_norm is None else k_norm.data_ptr(), T, B, N, page, cols, H, KH, hd, n, interleaved, q0, q1, k0, k1, v0,
                         v1, o0, o1, *pool, amplitude, eps, _raw_stream(dev))
    except (struct.error, OverflowError) as e:
        _no_number(e)
    _run(dev, record)
    _written((k_pages, v_pages) if k_scales is None else (k_pages, v_pages, k_scales, v_scales))
    if given:
        _written(out)
    return out


def _refuse_append(k, v, k_pages, v_pages, tables, lens, cu, k_scales, v_scales, freqs, positions, q, q_norm, k_norm, out):
    kinds, i32, f32 = tuple(_DTYPES), (torch.int32,), (torch.float32,)
    if not isinstance(k, torch.Tensor) or k.dim() != 3 or k.dtype not in kinds:
        _refuse(k, ("k", k, kinds, (-1, -1, -1)))
    if not isinstance(lens, torch.Tensor) or lens.dim() != 1:
        _refuse(k, ("lens", lens, i32, (-1,)))
    (T, KH, hd), B, same = k.shape, lens.shape[0], (k.dtype,)
    if cu is None and (T % B if B else T):
        raise ValueError(f"without cu there are as many tokens of each sequence; got {T} of {B}")
    if q is None and out is not None:
        raise ValueError("out is for q")
    _refuse(k, ("k", k, kinds, (T, KH, hd)), ("v", v, same, (T, KH, hd)), ("lens", lens, i32, (B,)),
            *_pool_named(k.dtype, k_pages, v_pages, tables, k_scales, v_scales, B, KH, hd),
            cu is not None and ("cu", cu, i32, (B + 1,)), positions is not None and ("positions", positions, i32, (T,)),
            freqs is not None and ("freqs", freqs, (torch.float64,), (-1,)), q is not None and ("q", q, same, (T, -1, hd)),
            out is not None and ("out", out, same, tuple(q.shape)),
            q_norm is not None and ("q_norm", q_norm, f32, (hd,)), k_norm is not None and ("k_norm", k_norm, f32, (hd,)))


def attention_paged(q, k_pages, v_pages, tables, lens, *, k_scales=None, v_scales=None, max_len=None, window=0, sinks=None,
                    scale=None, out=None):
    """The newest tokens of each sequence over its pages, causal.

    q [B, H, hd], one token each, or [B, n, H, hd], the n newest of each (a
    few drafted tokens; a whole prompt is faster through cache_gather and
    attention.attention_prompt); H a multiple of KH, up to 128 heads share a key
    head.  lens [B] int32: the positions of each sequence, its newest tokens'
    keys among them: query i of n is at lens - n + i and attends to the
    positions up to it, the last `window` of them if window > 0.  max_len: an
    upper bound of lens, if known (default: all that the tables hold); a larger
    value in lens counts as max_len.  sinks, scale: as attention.attention_prompt.
    A query without a key gives zeros.  Rows behind lens or before every
    query's window are not read, and nothing that a query does not attend to
    reaches it, infinities and NaN neither; a score of NaN or +inf among its keys
    makes its outputs NaN, one of -inf has no weight.  The softmax weights keep
    22 bits, with bfloat16 pages 16.  Over 8-bit pages bfloat16 queries are taken
    in fp16 times a power of two of their head's own: values below 2^-31 of the
    head's largest may lose bits, below 2^-40 they count as zero.  Returns out, of
    q's shape."""
    given = out is not None
    try:
        dtype, dev, shape = q.dtype, q.get_device(), q.shape
        kind = _DTYPES[dtype]
        if len(shape) == 4:
            (B, n, H, hd), (q0, q1, q2, q3) = shape, q.stride()
            if not given:
                out = _empty(shape, (max(n * H, 1) * hd, max(H, 1) * hd, hd, 1), dtype=dtype, device=q.device)
            o0, o1, o2, o3 = out.stride()
        else:
            (B, H, hd), (q0, q2, q3), n, q1, o1 = shape, q.stride(), 1, 8, 8
            if not given:
                out = _empty(shape, (H * hd, hd, 1), dtype=dtype, device=q.device)
            o0, o2, o3 = out.stride()
        N, KH, page, _ = k_pages.shape
        pool = _pool(dev, dtype, k_pages, v_pages, tables, k_scales, v_scales, KH, hd)
        rows, cols = tables.shape
        fit = (pool and dev >= 0 and q3 == o3 == 1 and rows == B and lens is not None and _vector(lens, dev, _I32, B)
               and (not given or (out.shape == shape and out.dtype is dtype and out.get_device() == dev))
               and (sinks is None or _vector(sinks, dev, _F32, H)))
    except _MISFITS:
        fit = False
    if not fit:
        _refuse_paged(q, k_pages, v_pages, tables, lens, k_scales, v_scales, sinks, out if given else None)
    if (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad or out.requires_grad
            or (k_scales is not None and (k_scales.requires_grad or v_scales.requires_grad)) or (sinks is not None and sinks.requires_grad)):
        _no_backward()
    if _forward._current_level >= 0:
        _no_tangents(q, k_pages, v_pages, k_scales, v_scales, sinks, out)
    most = cols * page
    try:
        max_len = most if max_len is None or max_len > most else max_len
        bits, window = 16 if k_scales is None else 8, _window(window)
        nbytes = load().tg_attention_paged_workspace(bits, B, n, max_len, window, H, KH, hd) if 0 < max_len < _MOST else 0
        ws = _empty((nbytes,), (1,), dtype=torch.uint8, device=q.device) if nbytes else None
        record = _ATTEND(2, kind, bits, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), 0 if k_scales is None else k_scales.data_ptr(),
                         0 if k_scales is None else v_scales.data_ptr(), out.data_ptr(), tables.data_ptr(), lens.data_ptr(),
                         0 if sinks is None else sinks.data_ptr(), B, n, N, page, cols, max_len, H, KH, hd, window, q0, q1, q2, o0, o1, o2,
                         *pool, hd ** -0.5 if scale is None else scale, 0 if ws is None else ws.data_ptr(), nbytes, _raw_stream(dev))
    except (struct.error, OverflowError, TypeError, ctypes.ArgumentError) as e:
        _no_number(e)
    _run(dev, record)
    if given:
        _written(out)
    return out


def _refuse_paged(q, k_pages, v_pages, tables, lens, k_scales, v_scales, sinks, out):
    kinds = tuple(_DTYPES)
    if not isinstance(q, torch.Tensor) or q.dim() not in (3, 4) or q.dtype not in kinds:
        _refuse(q, ("q", q, kinds, (-1, -1, -1)))
    B, H, hd = q.shape[0], q.shape[-2], q.shape[-1]
    _refuse(q, ("q", q, kinds, tuple(q.shape)), ("lens", lens, (torch.int32,), (B,)),
            *_pool_named(q.dtype, k_pages, v_pages, tables, k_scales, v_scales, B, -1, hd),
            sinks is not None and ("sinks", sinks, (torch.float32,), (H,)),
            out is not None and ("out", out, (q.dtype,), tuple(q.shape)))


def cache_gather(k_pages, v_pages, tables, cu, total, *, k_scales=None, v_scales=None, dtype=None, out=None):
    """The first positions of each sequence read back from its pages, packed.

    Sequence b's are the rows cu[b] .. cu[b + 1] (int32 on the device, B + 1
    ascending values) of the outputs [total, KH, hd], as attention.attention_prompt
    takes them with cu_k=cu.  dtype: the outputs' type for pages of 8 bits
    (bfloat16 unless out says otherwise); pages of 16 bits keep theirs.  Rows on a
    page outside the pool or behind the table read as zeros; rows of no
    sequence are not written.  out: (k, v) to write.  Returns (k, v)."""
    given = out is not None
    try:
        pages, dev, (N, KH, page, hd) = k_pages.dtype, k_pages.get_device(), k_pages.shape
        if dtype is None:
            dtype = out[0].dtype if given else torch.bfloat16 if pages is _CODES else pages
        kind, shape = _DTYPES[dtype], (total, KH, hd)
        if given:
            ko, vo = out
            (k0, k1, k2), (v0, v1, v2) = ko.stride(), vo.stride()
            fit = (ko.shape == vo.shape == shape and ko.dtype is vo.dtype is dtype and ko.get_device() == vo.get_device() == dev
                   and k2 == v2 == 1)
        else:
            k0, k1 = v0, v1 = strides = KH * hd, hd
            where = k_pages.device
            ko, vo = _empty(shape, (*strides, 1), dtype=dtype, device=where), _empty(shape, (*strides, 1), dtype=dtype, device=where)
            fit = True
        pool = _pool(dev, dtype, k_pages, v_pages, tables, k_scales, v_scales, KH, hd)
        B, cols = tables.shape
        fit = fit and pool and dev >= 0 and cu is not None and _vector(cu, dev, _I32, B + 1)
    except (*_MISFITS, RuntimeError):
        fit = False
    if not fit:
        _refuse_gather(k_pages, v_pages, tables, cu, total, k_scales, v_scales, dtype, out if given else None)
    if (k_pages.requires_grad or v_pages.requires_grad or ko.requires_grad or vo.requires_grad
            or (k_scales is not None and (k_scales.requires_grad or v_scales.requires_grad))):
        _no_backward()
    if _forward._current_level >= 0:
        _no_tangents(k_pages, v_pages, k_scales, v_scales, ko, vo)
    try:
        record = _GATHER(3, kind, 16 if k_scales is None else 8, k_pages.data_ptr(), v_pages.data_ptr(),
                         0 if k_scales is None else k_scales.data_ptr(), 0 if k_scales is None else v_scales.data_ptr(), tables.data_ptr(),
                         cu.data_ptr(), ko.data_ptr(), vo.data_ptr(), total, B, N, page, cols, KH, hd, k0, k1, v0, v1, *pool, _raw_stream(dev))
    except (struct.error, OverflowError) as e:
        _no_number(e)
    _run(dev, record)
    if given:
        _written(ko)
        _written(vo)
    return ko, vo


def _refuse_gather(k_pages, v_pages, tables, cu, total, k_scales, v_scales, dtype, out):
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() != 4:
        _refuse(k_pages, ("k_pages", k_pages, (*_DTYPES, _CODES), (-1, -1, -1, -1)))
    if not isinstance(total, int) or total < 0:
        raise ValueError(f"total must be a number of rows; is {total!r}")
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be bfloat16 or float16; is {dtype}")
    if k_pages.dtype not in (dtype, _CODES):
        raise ValueError(f"pages of {k_pages.dtype} are not read as {dtype}")
    KH, hd = k_pages.shape[1], k_pages.shape[3]
    B = tables.shape[0] if isinstance(tables, torch.Tensor) and tables.dim() else -1
    ko, vo = (None, None) if out is None else out if isinstance(out, (tuple, list)) and len(out) == 2 else (out, out)
    _refuse(k_pages, *_pool_named(dtype, k_pages, v_pages, tables, k_scales, v_scales, B, KH, hd),
            ("cu", cu, (torch.int32,), (B + 1,)), out is not None and ("out[0]", ko, (dtype,), (total, KH, hd)),
            out is not None and ("out[1]", vo, (dtype,), (total, KH, hd)))
