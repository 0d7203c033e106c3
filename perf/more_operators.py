"""A paged key/value cache and what a server does with it next to the mixture-of-experts layers: the work it is measured on.

Four operators on device tensors (tinygiant_b200.paged):

  rotary   queries and keys rotated by their positions, halves or neighbours paired, part of a head or all of it, frequencies
           scaled for long contexts, with the norm of each head before;
  append   new tokens' keys, rotated on the way, and values written to their pages: in 16 bits, or in 8 with a scale for each
           block of 16 tokens and head; the queries rotated in the same call;
  paged    the newest tokens of each sequence attend to its pages, with sliding windows and per-head sink logits;
  gather   pages read back as packed 16-bit keys and values, for the attention of a prompt that arrives in chunks.

`own` chooses between the plain torch form and the calls of the package.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 16                                                       # tokens under one scale
LOW = -117                                                       # exponent of the smallest scale


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _spread(n, low, high, step=7919):
    """n odd-sized lengths between low and high, the same each time."""
    return [low + (i * step + 13) % (high - low + 1) for i in range(n)]


def _rope(kind="plain", rot=128, theta=1e6, factor=1.0, interleaved=False, norms=True):
    return {"rope": kind, "rot": rot, "theta": theta, "factor": factor, "interleaved": interleaved, "norms": norms}


def _rotary(name, dtype, heads, kv_heads, head_dim, tokens, first, rope):
    """tokens: rows, at positions from `first` on."""
    return {"name": name, "op": "rotary", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "tokens": tokens, "first": first, **rope}


def _append(name, dtype, bits, heads, kv_heads, head_dim, page, lens, ctx, rope):
    """lens: new tokens of each sequence; ctx: tokens of each that the cache holds before."""
    return {"name": name, "op": "append", "dtype": dtype, "bits": bits, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "lens": _text(lens), "ctx": _text(ctx), **rope}


def _paged(name, dtype, bits, heads, kv_heads, head_dim, page, new, lens, window=0, sinks=False):
    """new: queries of each sequence; lens: cached positions of each, its newest among them."""
    return {"name": name, "op": "paged", "dtype": dtype, "bits": bits, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "new": new, "lens": _text(lens), "window": window, "sinks": sinks}


def _gather(name, dtype, bits, kv_heads, head_dim, page, lens):
    return {"name": name, "op": "gather", "dtype": dtype, "bits": bits, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "lens": _text(lens)}


def listed():
    gptoss = _rope("yarn", 64, 150000.0, 32.0, norms=False)
    return [
        # a chunk of three tokens; latency
        _rotary("rotary_few_tokens", "bf16", 32, 4, 128, 3, 4089, _rope()),
        # a long prompt far into a context that was stretched 32 times, neighbours paired, half of each head
        _rotary("rotary_8192_far", "fp16", 32, 4, 128, 8192, 122880, _rope("yarn", 64, 150000.0, 32.0, True, False)),
        # two sequences' next tokens, one of them the first of a page; latency
        _append("append_pair", "bf16", 8, 32, 4, 128, 64, [1, 1], [32, 57], _rope()),
        # an odd batch that checks four drafted tokens each, in 16 bits
        _append("append_drafts_33", "fp16", 16, 64, 8, 64, 16, [4] * 33, _spread(33, 0, 50), gptoss),
        # chunks of requests of everyday sizes, one of them empty, behind what came before
        _append("append_ragged", "bf16", 8, 32, 4, 128, 16, [517, 1, 0, 1023, 77, 300, 129, 1],
                [0, 40, 19, 7, 512, 333, 5, 1000], _rope()),
        # the largest: one long prompt
        _append("append_8192", "bf16", 8, 32, 4, 128, 64, [8192], [0], _rope()),
        # two short sequences; latency
        _paged("paged_pair", "bf16", 8, 32, 4, 128, 64, 1, [100, 33]),
        # 64 heads of 64 with sinks and a window of 128, four drafted tokens each, an odd batch in 16 bits, one of it empty
        _paged("paged_window_sinks_33", "fp16", 16, 64, 8, 64, 16, 4, [0] + _spread(32, 4, 4096), 128, True),
        # an ordinary batch of everyday lengths
        _paged("paged_batch_64", "bf16", 8, 32, 4, 128, 16, 1, _spread(64, 1, 4096)),
        # the largest: a full batch of long contexts
        _paged("paged_batch_256", "bf16", 8, 32, 4, 128, 64, 1, _spread(256, 2048, 8192)),
        # an odd batch's earlier chunks, in small pages
        _gather("gather_ragged", "fp16", 8, 8, 64, 16, [517, 1, 0, 1023, 77, 300, 129, 1]),
        # the largest: what eight long documents have so far
        _gather("gather_8_of_8192", "bf16", 8, 4, 128, 64, [8192] * 6 + [8191, 5003]),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = [(32, 4), (64, 8), (16, 16), (8, 2), (28, 4), (24, 8), (16, 1)]


def draw(rng):
    op = rng.choice(["rotary", "append", "paged", "paged", "gather"])
    dtype = rng.choice(["bf16", "fp16"])
    bits = rng.choice([8, 8, 16])
    heads, kv_heads = rng.choice(HEADS)
    hd = rng.choice([64, 64, 80, 96, 128, 128, 128])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    most = {o: max(work(c)["bytes"] for c in listed() if c["op"] == o) for o in ("rotary", "append", "paged", "gather")}
    while True:
        kind = rng.choice(["plain", "plain", "linear", "ntk", "yarn"])
        rope = _rope(kind, rng.choice([hd, hd, hd // 2, hd // 4]), rng.choice([10000.0, 150000.0, 1e6]),
                     1.0 if kind == "plain" else float(rng.choice([2, 4, 8, 32])), rng.random() < 0.3, rng.random() < 0.5)
        if op == "rotary":
            case = _rotary("", dtype, heads, kv_heads, hd, _log(rng, 1, 8192), _log(rng, 1, 131072) - 1, rope)
        elif op == "append":
            n = _log(rng, 1, 64)
            few = rng.random() < 0.5
            lens = [rng.randint(0, 8) if few else _log(rng, 1, 8192) for _ in range(n)]
            lens[0] = max(1, lens[0])
            ctx = [_log(rng, 1, 2048) - 1 for _ in range(n)]
            case = _append("", dtype, bits, heads, kv_heads, hd, page, lens, ctx, rope)
        elif op == "paged":
            new, top = rng.choice([1, 1, 1, 2, 4, 8]), _log(rng, 8, 16384)
            lens = [rng.randint(0, top) for _ in range(_log(rng, 1, 256))]
            lens[0] = max(new, lens[0])
            case = _paged("", dtype, bits, heads, kv_heads, hd, page, new, lens, rng.choice([0, 0, 0, 128, 1000]),
                          rng.random() < 0.3)
        else:
            case = _gather("", dtype, bits, kv_heads, hd, page, [_log(rng, 1, 8192) - 1 for _ in range(_log(rng, 1, 16))] + [9])
        cells = len(_ints(case["lens"])) * max(_ints(case["lens"])) if op == "paged" else 0
        if work(case)["bytes"] <= most[op] and cells * kv_heads * hd <= 256 * 8192 * 4 * 128 and cells * heads * case.get("new", 1) <= 1 << 28:
            case.pop("name")
            return case


def work(case):
    hd, KH = case["head_dim"], case["kv_heads"]
    if case["op"] == "rotary":
        rows = case["tokens"] * (case["heads"] + KH)
        return {"bytes": 4 * rows * hd + 4 * case["tokens"] + 4 * case["rot"] + (8 * hd if case["norms"] else 0),
                "flops": rows * (3 * case["rot"] + (4 * hd if case["norms"] else 0))}
    per = case["bits"] // 8                                      # bytes of a cached value
    lens = _ints(case["lens"])
    scale = lambda n: 4 * -(-n // BLOCK) if per == 1 else 0      # noqa: E731  of the blocks of n tokens
    if case["op"] == "append":
        ctx, n = _ints(case["ctx"]), sum(lens)
        rows = n * (case["heads"] + KH)
        moved = 4 * n * case["heads"] * hd + 2 * KH * n * hd * (2 + per) + sum(2 * KH * scale(m) for m in lens)
        if per == 1:                                             # and all that the sequences have read back
            moved += sum(2 * KH * (3 * hd * (m + c) + scale(m + c)) for m, c in zip(lens, ctx))
        return {"bytes": moved + 8 * len(lens) + 4 * case["rot"],
                "flops": rows * (3 * case["rot"] + (4 * hd if case["norms"] else 0))}
    if case["op"] == "gather":
        return {"bytes": sum(2 * KH * (hd * (per + 2) * n + scale(n)) for n in lens) + 4 * len(lens), "flops": 0}
    H, new, window = case["heads"], case["new"], case["window"]
    moved = pairs = 0
    for n in lens:
        first = max(0, max(0, n - new) + 1 - window) if window else 0
        moved += 2 * KH * (hd * per * (n - first) + scale(n - first))
        for p in range(max(0, n - new), n):
            pairs += min(p + 1, window) if window else p + 1
    return {"bytes": moved + 4 * len(lens) * new * H * hd + 4 * len(lens) + (4 * H if case["sinks"] else 0), "flops": 4 * hd * H * pairs}


def _frequencies(case, dev):
    """Angles per position, fp64, and what the rotated values are multiplied by."""
    d, theta, factor = case["rot"], case["theta"], case["factor"]
    if case["rope"] == "ntk":
        theta *= factor ** (d / (d - 2))
    f = [theta ** (-2 * j / d) for j in range(d // 2)]
    if case["rope"] == "linear":
        f = [x / factor for x in f]
    if case["rope"] == "yarn":
        turn = lambda n: d * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(turn(32)), 0), min(math.ceil(turn(1)), d - 1)
        keep = [1 - min(1, max(0, (j - low) / max(high - low, 0.001))) for j in range(d // 2)]
        f = [x * k + x / factor * (1 - k) for x, k in zip(f, keep)]
    return torch.tensor(f, dtype=torch.float64, device=dev), 0.1 * math.log(factor) + 1 if case["rope"] == "yarn" else 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, hd, KH = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]
    dev = torch.device("cuda")

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    s = {"op": case["op"], "dtype": dt}
    if case["op"] in ("rotary", "append"):
        s["freqs"], s["amplitude"] = _frequencies(case, dev)
        s["interleaved"] = case["interleaved"]
        s["q_norm"] = s["k_norm"] = None
        if case["norms"]:
            s["q_norm"], s["k_norm"] = (1 + 0.2 * torch.randn(hd, generator=g, device=dev) for _ in range(2))
    if case["op"] == "rotary":
        n = case["tokens"]
        # as they come from one product
        qkv = normal(n, case["heads"] + 2 * KH, hd, scale=1.5)
        s["q"], s["k"] = qkv[:, :case["heads"]], qkv[:, case["heads"]:case["heads"] + KH]
        s["positions"] = case["first"] + torch.arange(n, dtype=torch.int32, device=dev)
        return s
    lens, ps = _ints(case["lens"]), case["page"]
    ctx = _ints(case["ctx"]) if case["op"] == "append" else [0] * len(lens)
    ends = [a + b for a, b in zip(lens, ctx)]
    # pages of a pool in any order; a sequence's pages behind its end are none
    need = [-(-n // ps) for n in ends]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device=dev).int().tolist()
    tables, at = [], 0
    for n in need:
        tables.append(order[at:at + n] + [-1] * (max(need) - n))
        at += n
    s["tables"] = torch.tensor(tables, dtype=torch.int32, device=dev)
    s["lens"] = torch.tensor(ends, dtype=torch.int32, device=dev)
    total = lambda ns: torch.tensor([sum(ns[:i]) for i in range(len(ns) + 1)], dtype=torch.int32, device=dev)  # noqa: E731
    s["cu"] = total(ends if case["op"] == "gather" else lens)
    s["total"], s["max_len"] = sum(ends), max(ends)
    # keys of a few wide channels, values of tokens that differ
    wide = torch.exp(0.5 * torch.randn(hd, generator=g, device=dev))
    for x in "kv":
        if case["bits"] == 16:
            s[x + "_pages"], s[x + "_scales"] = torch.empty(pool, KH, ps, hd, dtype=dt, device=dev), None
        else:
            s[x + "_pages"] = torch.empty(pool, KH, ps, hd, dtype=torch.float8_e4m3fn, device=dev)
            s[x + "_scales"] = torch.empty(pool, KH, ps // BLOCK, device=dev)
        step = max(1, (1 << 27) // (KH * ps * hd))
        for i in range(0, pool, step):
            n = min(step, pool - i)
            y = torch.randn(n, KH, ps // BLOCK, BLOCK, hd, generator=g, device=dev)
            y *= wide if x == "k" else torch.exp(0.5 * torch.randn(n, KH, ps // BLOCK, 1, 1, generator=g, device=dev))
            if case["bits"] == 16:
                s[x + "_pages"][i:i + n] = y.view(n, KH, ps, hd).to(dt)
            else:
                scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax((3, 4)) / 448)))
                s[x + "_pages"][i:i + n] = (y / scale[..., None, None]).view(n, KH, ps, hd).to(torch.float8_e4m3fn)
                s[x + "_scales"][i:i + n] = scale
    if case["op"] == "append":
        qkv = normal(sum(lens), case["heads"] + 2 * KH, hd, scale=1.5)
        s["q"], s["k"], s["v"] = qkv.split([case["heads"], KH, KH], 1)
    if case["op"] == "paged":
        q = normal(len(lens), case["new"], case["heads"], hd, scale=1.5)
        s["q"] = q if case["new"] > 1 else q[:, 0]
        s["window"] = case["window"]
        s["sinks"] = torch.randn(case["heads"], generator=g, device=dev) if case["sinks"] else None
    return s


def run(state):
    s = state
    if own:
        from tinygiant_b200 import paged as P
        if s["op"] == "rotary":
            return P.rotary(s["q"], s["k"], s["positions"], s["freqs"], interleaved=s["interleaved"], amplitude=s["amplitude"],
                            q_norm=s["q_norm"], k_norm=s["k_norm"])
        scales = {"k_scales": s["k_scales"], "v_scales": s["v_scales"]}
        if s["op"] == "append":
            q = P.cache_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], s["cu"], **scales,
                               freqs=s["freqs"], interleaved=s["interleaved"], amplitude=s["amplitude"], q=s["q"],
                               q_norm=s["q_norm"], k_norm=s["k_norm"])
            if s["k_scales"] is None:
                return q, s["k_pages"], s["v_pages"]
            cu = torch.nn.functional.pad(torch.cumsum(s["lens"], 0, dtype=torch.int32), (1, 0))
            return (q, *P.cache_gather(s["k_pages"], s["v_pages"], s["tables"], cu, s["total"], **scales, dtype=s["dtype"]))
        if s["op"] == "paged":
            return P.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], **scales, max_len=s["max_len"],
                                     window=s["window"], sinks=s["sinks"])
        return P.cache_gather(s["k_pages"], s["v_pages"], s["tables"], s["cu"], s["total"], **scales, dtype=s["dtype"])
    if s["op"] == "rotary":
        return (_plain_rotate(s["q"], s["positions"], s, s["q_norm"]).to(s["dtype"]),
                _plain_rotate(s["k"], s["positions"], s, s["k_norm"]).to(s["dtype"]))
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "paged":
        return _plain_paged(s)
    return _plain_gather(s, s["cu"])


def _plain_rotate(x, positions, s, norm):
    x = x.float()
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * norm
    d = 2 * len(s["freqs"])
    angle = positions.double()[:, None] * s["freqs"]
    c, n = (torch.cos(angle) * s["amplitude"]).float()[:, None], (torch.sin(angle) * s["amplitude"]).float()[:, None]
    if s["interleaved"]:
        a, b = x[..., :d:2], x[..., 1:d:2]
        y = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = x[..., :d // 2], x[..., d // 2:d]
        y = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([y, x[..., d:]], -1)


def _plain_scale(amax):
    """The least power of two under which amax fits e4m3's 448 = 1.75 x 2^8."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e - 8 - (m <= 0.875).int(), LOW).clamp(min=LOW))


def _plain_append(s):
    """Tokens to their places; in 8 bits block by block, with the blocks that have earlier tokens rounded again where their scale grows."""
    (T, KH, hd), ps, dev = s["k"].shape, s["k_pages"].shape[2], s["k"].device
    seq = torch.searchsorted(s["cu"], torch.arange(T, dtype=torch.int32, device=dev), right=True) - 1
    pos = torch.arange(T, device=dev) - s["cu"][seq + 1] + s["lens"][seq]
    page, row = s["tables"][seq, pos // ps].long(), pos % ps
    q = _plain_rotate(s["q"], pos, s, s["q_norm"]).to(s["dtype"])
    new = {"k": _plain_rotate(s["k"], pos, s, s["k_norm"]), "v": s["v"].float()}
    if s["k_scales"] is None:
        for x in "kv":
            s[x + "_pages"][page, :, row] = new[x].to(s["dtype"])
        return q, s["k_pages"], s["v_pages"]
    bpp = ps // BLOCK
    block = page * bpp + row // BLOCK                            # of each new token, among the pool's
    # the block of each sequence's first new token, where it has rows from before; the others have one behind the pool's
    none = s["k_scales"].numel() // KH
    first = s["lens"] - (s["cu"][1:] - s["cu"][:-1])
    old_rows = torch.where(s["cu"][1:] > s["cu"][:-1], first % BLOCK, 0)
    old_page = s["tables"].gather(1, torch.clamp(first // ps, max=s["tables"].shape[1] - 1).long()[:, None])[:, 0].long()
    old = torch.where(old_rows > 0, old_page * bpp + first % ps // BLOCK, none)                  # [B]
    r = torch.arange(BLOCK, device=dev)
    seq_r, r = (r < old_rows[:, None]).nonzero(as_tuple=True)    # the rows from before: their sequence, and row of the block
    at = old_page[seq_r], first[seq_r] % ps // BLOCK * BLOCK + r
    for x in "kv":
        pages, scales = s[x + "_pages"], s[x + "_scales"]
        kept = torch.nn.functional.pad(scales.transpose(1, 2).reshape(-1, KH), (0, 0, 0, 1))[old]                 # [B, KH]
        amax = torch.zeros(none + 1, KH, device=dev)
        amax.scatter_reduce_(0, block[:, None].expand(T, KH), new[x].abs().amax(-1), "amax")
        scale = _plain_scale(amax)
        scale[old] = torch.maximum(scale[old], kept)
        ratio = (kept / scale[old])[seq_r][..., None]
        pages.view(torch.uint8)[at[0], :, at[1]] = (pages[at[0], :, at[1]].float() * ratio).to(pages.dtype).view(torch.uint8)
        pages.view(torch.uint8)[page, :, row] = (new[x] / scale[block][..., None]).to(pages.dtype).view(torch.uint8)
        scales[page, :, row // BLOCK] = scale[block]
    return (q, *_plain_gather(s, torch.nn.functional.pad(torch.cumsum(s["lens"], 0, dtype=torch.int32), (1, 0))))


def _plain_values(s, x, page, row):
    """Values of the cache's rows, [.., KH, hd] in fp32."""
    y = s[x + "_pages"][page, :, row].float()
    return y if s[x + "_scales"] is None else y * s[x + "_scales"][page, :, row // BLOCK][..., None]


def _plain_gather(s, cu):
    i = torch.arange(s["total"], dtype=torch.int32, device=cu.device)
    seq = torch.searchsorted(cu, i, right=True) - 1
    pos, ps = i - cu[seq], s["k_pages"].shape[2]
    page = s["tables"][seq, pos // ps].long()
    return tuple(_plain_values(s, x, page, pos % ps).to(s["dtype"]) for x in "kv")


def _plain_paged(s):
    q = s["q"].float()
    q = q if q.dim() == 4 else q[:, None]
    (B, n, H, hd), KH, ps, L, dev = q.shape, s["k_pages"].shape[1], s["k_pages"].shape[2], s["max_len"], q.device
    j = torch.arange(L, device=dev)
    there = j < s["lens"][:, None]                               # [B, L]
    page = torch.where(there, s["tables"][:, :-(-L // ps)].long().repeat_interleave(ps, 1)[:, :L], 0)
    k, v = (_plain_values(s, x, page, (j % ps).expand(B, L)).masked_fill_(~there[..., None, None], 0.0) for x in "kv")
    pos = s["lens"][:, None] - n + torch.arange(n, device=dev)   # [B, n]
    gone = j > pos[..., None]
    if s["window"]:
        gone |= j <= pos[..., None] - s["window"]
    qs = (q / math.sqrt(hd)).view(B, n, KH, H // KH, hd).permute(0, 2, 1, 3, 4).reshape(B, KH, n * (H // KH), hd)
    scores = torch.matmul(qs, k.permute(0, 2, 3, 1)).view(B, KH, n, H // KH, L)
    scores.masked_fill_(gone[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    sinks = None if s["sinks"] is None else s["sinks"].view(KH, 1, H // KH, 1)
    top = top if sinks is None else torch.maximum(top, sinks)
    top = torch.where(top == -math.inf, 0.0, top)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    total = total if sinks is None else total + torch.exp(sinks - top)
    o = torch.matmul(scores.view(B, KH, -1, L), v.transpose(1, 2)).view(B, KH, n, H // KH, hd)
    o = (o * torch.where(total == 0, 0.0, 1 / total)).permute(0, 2, 1, 3, 4).reshape(B, n, H, hd).to(s["dtype"])
    return o if s["q"].dim() == 4 else o[:, 0]


def _grid(y):
    """The nearest number of e4m3, even at ties, for |y| <= 448."""
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -30))), min=-6) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    """From the definitions, sequence by sequence, in 64 bits."""
    s = prepare(case, seed)
    hd, KH = case["head_dim"], case["kv_heads"]

    def rotated(x, positions, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + 1e-6) * w.double()
        y, d = x.clone(), case["rot"]
        for j in range(d // 2):
            a, b = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + d // 2)
            t = (positions.double() * s["freqs"][j])[:, None]
            y[..., a] = s["amplitude"] * (x[..., a] * torch.cos(t) - x[..., b] * torch.sin(t))
            y[..., b] = s["amplitude"] * (x[..., b] * torch.cos(t) + x[..., a] * torch.sin(t))
        return y

    if s["op"] == "rotary":
        return rotated(s["q"], s["positions"], s["q_norm"]), rotated(s["k"], s["positions"], s["k_norm"])
    lens, ps, tables = _ints(case["lens"]), case["page"], s["tables"].tolist()

    def held(x, b, n):
        """The first n positions of sequence b, [n, KH, hd]."""
        parts = [torch.zeros(0, KH, hd, dtype=torch.float64, device=s["k_pages"].device)]
        for i in range(-(-n // ps)):
            y = s[x + "_pages"][tables[b][i]].double()
            if case["bits"] == 8:
                y = y * s[x + "_scales"][tables[b][i]].double().repeat_interleave(BLOCK, 1)[..., None]
            parts.append(y.transpose(0, 1))
        return torch.cat(parts)[:n]

    if s["op"] == "gather":
        return tuple(torch.cat([held(x, b, n) for b, n in enumerate(lens)]) for x in "kv")
    if s["op"] == "append":
        ctx, cu = _ints(case["ctx"]), [sum(lens[:i]) for i in range(len(lens) + 1)]
        pos = torch.cat([torch.arange(c, c + n, device=s["k"].device) for n, c in zip(lens, ctx)])
        q, new = rotated(s["q"], pos, s["q_norm"]), {"k": rotated(s["k"], pos, s["k_norm"]), "v": s["v"].double()}
        if case["bits"] == 16:
            out = {x: s[x + "_pages"].double() for x in "kv"}
            for x in "kv":
                for b, (n, c) in enumerate(zip(lens, ctx)):
                    for i in range(c // ps, -(-(c + n) // ps)):
                        lo, hi = max(c, i * ps), min(c + n, (i + 1) * ps)
                        out[x][tables[b][i], :, lo - i * ps:hi - i * ps] = new[x][cu[b] + lo - c:cu[b] + hi - c].transpose(0, 1)
            return q, out["k"], out["v"]
        back = {"k": [], "v": []}
        for x in "kv":
            for b, (n, c) in enumerate(zip(lens, ctx)):
                y = torch.cat([held(x, b, c), new[x][cu[b]:cu[b + 1]]])
                for lo in range(c // BLOCK * BLOCK, c + n if n else 0, BLOCK):
                    part = y[max(lo, c):lo + BLOCK]
                    need = part.abs().amax((0, 2)) / 448
                    scale = torch.exp2(torch.ceil(torch.log2(torch.clamp(need, min=2.0 ** LOW))))     # [KH]
                    if lo < c:
                        old = s[x + "_scales"][tables[b][lo // ps], :, lo % ps // BLOCK].double()
                        scale = torch.maximum(scale, old)
                    y[lo:lo + BLOCK] = _grid(y[lo:lo + BLOCK] / scale[:, None]) * scale[:, None]
                back[x].append(y)
        return q, torch.cat(back["k"]), torch.cat(back["v"])
    H, new, window = case["heads"], case["new"], case["window"]
    q = s["q"].double()
    q = q if q.dim() == 4 else q[:, None]
    out = torch.zeros_like(q)
    for b, n in enumerate(lens):
        k, v = held("k", b, n), held("v", b, n)
        for i in range(new):
            p = n - new + i
            if p < 0:
                continue
            lo = max(0, p + 1 - window) if window else 0
            kk, vv = k[lo:p + 1].transpose(0, 1), v[lo:p + 1].transpose(0, 1)                         # [KH, keys, hd]
            x = torch.matmul(q[b, i].view(KH, H // KH, hd), kk.transpose(1, 2)) / math.sqrt(hd)
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"].double().view(KH, H // KH, 1)], 2)
            w = torch.softmax(x, 2)[..., :p + 1 - lo]
            out[b, i] = torch.matmul(w, vv).view(H, hd)
    return out if s["q"].dim() == 4 else out[:, 0]
