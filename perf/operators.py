"""Attention over a key/value cache, as a server runs it next to the mixture-of-experts layers: the work it is measured on.

Three operators on device tensors (tinygiant_b200.attention):

  prompt   causal attention of whole prompts packed one after another, grouped query heads, with a sliding window, per-head
           sink logits and keys that are there before the prompt's own (a prompt that arrives in chunks);
  shared   one token of each sequence of a batch against a prefix that all of them share and each one's own cache, adding the
           attention that every cached key got to a running weight;
  evict    the cache cut down to a budget: the newest positions and the heaviest of the others stay, moved together.

`own` chooses between the plain torch form and the calls of the package.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _prompt(name, dtype, heads, kv_heads, head_dim, lens, ctx=None, window=0, sinks=False):
    """lens: new tokens of each sequence; ctx: keys of each that were there before."""
    ctx = [0] * len(lens) if ctx is None else ctx
    return {"name": name, "op": "prompt", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "lens": _text(lens), "ctx": _text(ctx), "window": window, "sinks": sinks}


def _shared(name, dtype, heads, kv_heads, head_dim, prefix, cap, lens, window=0, sinks=False, weights=True):
    """lens: own cached positions of each sequence, its newest token's among them; cap: rows of each one's cache."""
    return {"name": name, "op": "shared", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "prefix": prefix, "cap": cap, "lens": _text(lens), "window": window, "sinks": sinks, "weights": weights}


def _evict(name, dtype, kv_heads, head_dim, cap, lens, keep, recent):
    return {"name": name, "op": "evict", "dtype": dtype, "kv_heads": kv_heads, "head_dim": head_dim, "cap": cap,
            "lens": _text(lens), "keep": keep, "recent": recent}


def _spread(n, low, high, step=7919):
    """n odd-sized lengths between low and high, the same each time."""
    return [low + (i * step + 13) % (high - low + 1) for i in range(n)]


def listed():
    return [
        # the engine's smallest calls: a chunk of eight tokens and less, three requests at once; latency
        _prompt("prompt_few_tokens", "bf16", 32, 4, 128, [8, 1, 5]),
        # the last chunk of eight of a prompt that fills the engine's default cache: few rows, a long axis
        _prompt("prompt_chunk_on_4088", "bf16", 32, 4, 128, [8], [4088]),
        # requests of everyday sizes in one pass, one of them empty, none a multiple of anything
        _prompt("prompt_ragged", "fp16", 32, 4, 128, [517, 1, 0, 1023, 77, 300, 129, 1]),
        # 64 heads of 64 with sinks and a window of 128, as every other layer of such a model has it
        _prompt("prompt_window_sinks", "bf16", 64, 8, 64, [2048, 701, 1347], window=128, sinks=True),
        # the largest: one long prompt
        _prompt("prompt_8192", "bf16", 32, 4, 128, [8192]),
        # a pair of sequences on a short system prompt; latency
        _shared("shared_pair", "bf16", 32, 4, 128, 100, 64, [17, 33]),
        # an ordinary batch on a long system prompt, weights kept for a later eviction
        _shared("shared_batch_64", "bf16", 32, 4, 128, 4096, 640, _spread(64, 1, 640)),
        # 64 heads of 64 with sinks, an odd batch, one sequence that has no key of its own yet
        _shared("shared_sinks_33", "fp16", 64, 8, 64, 1531, 2048, [0] + _spread(32, 1, 2048), sinks=True, weights=False),
        # the largest: a full batch on a document that all of them ask about
        _shared("shared_batch_256", "bf16", 32, 4, 128, 16384, 1024, _spread(256, 512, 1024)),
        # two sequences just over their budget; latency
        _evict("evict_pair", "bf16", 4, 128, 300, [300, 257], 256, 32),
        # an odd batch of odd lengths, some of them under the budget
        _evict("evict_ragged", "fp16", 8, 64, 4096, _spread(13, 100, 4096), 1000, 100),
        # the largest: long prompts cut to a quarter for decoding
        _evict("evict_8192", "bf16", 8, 128, 8192, [8192] * 24 + [8191, 7000, 8192, 5003, 8000, 8192, 4097, 8192], 2048, 256),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = [(32, 4), (64, 8), (16, 16), (8, 2), (28, 4), (24, 8), (16, 1)]


def draw(rng):
    op = rng.choice(["prompt", "shared", "evict"])
    dtype = rng.choice(["bf16", "fp16"])
    heads, kv_heads = rng.choice(HEADS)
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128])
    top = max(work(c)["flops"] for c in listed() if c["op"] == "prompt")
    most = {o: max(work(c)["bytes"] for c in listed() if c["op"] == o) for o in ("shared", "evict")}
    while True:
        if op == "prompt":
            n = _log(rng, 1, 16)
            lens = [_log(rng, 1, 8192) if rng.random() > 0.05 else 0 for _ in range(n)]
            ctx = [_log(rng, 1, 8192) if rng.random() < 0.3 else 0 for _ in range(n)]
            window = rng.choice([0, 0, 0, 128, 1000])
            case = _prompt("", dtype, heads, kv_heads, head_dim, lens, ctx, window, rng.random() < 0.3)
            tq, tk = sum(lens), sum(lens) + sum(ctx)
            fits = 0 < tq and heads * tq * tk <= 32 * 8192 * 8192 and work(case)["flops"] <= top
        elif op == "shared":
            n, cap = _log(rng, 1, 256), _log(rng, 16, 8192)
            lens = [rng.randint(0, cap) for _ in range(n)]
            prefix = _log(rng, 1, 16384) if rng.random() > 0.05 else 0
            window = rng.choice([0, 0, 0, 0, 128, 4096])
            case = _shared("", dtype, heads, kv_heads, head_dim, prefix, cap, lens, window, rng.random() < 0.3,
                           rng.random() < 0.6)
            w = work(case)
            fits = (n * kv_heads * cap * head_dim <= 256 * 4 * 1024 * 128 and n * heads * (prefix + cap) <= 1 << 28
                    and w["bytes"] <= most[op] and w["flops"] <= top)
        else:
            n, cap = _log(rng, 1, 64), _log(rng, 16, 16384)
            lens = [rng.randint(0, cap) if rng.random() < 0.5 else cap for _ in range(n)]
            keep = max(1, min(cap, int(cap * rng.uniform(0.1, 0.9))))
            case = _evict("", dtype, kv_heads, head_dim, cap, lens, keep, rng.randint(0, keep))
            fits = n * kv_heads * cap * head_dim <= 32 * 8 * 8192 * 128 and work(case)["bytes"] <= most[op]
        if fits:
            case.pop("name")
            return case


def work(case):
    hd, es = case["head_dim"], 2
    if case["op"] == "prompt":
        H, KH, window = case["heads"], case["kv_heads"], case["window"]
        pairs = rows = keys = 0
        for n, c in zip(_ints(case["lens"]), _ints(case["ctx"])):
            if n == 0:
                continue
            w = window or n + c
            full = max(0, min(n, n + c - w))                     # rows that see w keys
            rest = n - full                                      # rows that see c + 1, c + 2, ... keys
            pairs += full * w + rest * c + rest * (rest + 1) // 2
            rows += n
            keys += min(n + c, n - 1 + w)
        return {"bytes": es * hd * (2 * rows * H + 2 * keys * KH) + (4 * H if case["sinks"] else 0),
                "flops": 4 * hd * H * pairs}
    if case["op"] == "shared":
        H, KH, P, window = case["heads"], case["kv_heads"], case["prefix"], case["window"]
        lens = _ints(case["lens"])
        own_keys = sum(min(n, window) if window else n for n in lens)
        pre = [min(P, max(0, window - n)) if window else P for n in lens]
        bytes_ = es * hd * (2 * len(lens) * H + 2 * max(pre) * KH + 2 * own_keys * KH) + 4 * len(lens)
        if case["weights"]:
            bytes_ += 8 * own_keys * KH
        return {"bytes": bytes_ + (4 * H if case["sinks"] else 0), "flops": 4 * hd * H * (sum(pre) + own_keys)}
    KH, keep = case["kv_heads"], case["keep"]
    lens = _ints(case["lens"])
    kept = sum(min(n, keep) for n in lens)
    scored = sum(n for n in lens if n > keep)
    out_rows = len(lens) * keep
    return {"bytes": KH * (2 * es * hd * (kept + out_rows) + 4 * (scored + kept) + 8 * out_rows) + 8 * len(lens), "flops": 0}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, hd = DTYPES[case["dtype"]], case["head_dim"]
    dev = torch.device("cuda")

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    lens = _ints(case["lens"])
    s = {"op": case["op"]}
    if case["op"] == "evict":
        KH, cap = case["kv_heads"], case["cap"]
        s["k"], s["v"] = normal(len(lens), KH, cap, hd), normal(len(lens), KH, cap, hd)
        # few keys get most of the attention, and some got none at all
        w = torch.exp(1.5 * torch.randn(len(lens), KH, cap, generator=g, device=dev))
        s["weights"] = w * (torch.rand(len(lens), KH, cap, generator=g, device=dev) > 0.1)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["keep"], s["recent"] = case["keep"], case["recent"]
        return s
    H, KH = case["heads"], case["kv_heads"]
    s["window"] = case["window"]
    s["sinks"] = torch.randn(H, generator=g, device=dev) if case["sinks"] else None
    if case["op"] == "prompt":
        ctx = _ints(case["ctx"])
        tq, tk = sum(lens), sum(lens) + sum(ctx)
        # queries and keys after their norms: scores a little wider than a unit normal
        s["q"], s["k"], s["v"] = normal(tq, H, hd, scale=1.5), normal(tk, KH, hd), normal(tk, KH, hd, scale=0.7)
        ends = lambda ns: torch.tensor([sum(ns[:i]) for i in range(len(ns) + 1)], dtype=torch.int32, device=dev)  # noqa: E731
        s["cu_q"], s["cu_k"] = ends(lens), ends([a + b for a, b in zip(lens, ctx)])
        s["max_k"] = max(a + b for a, b in zip(lens, ctx))
        return s
    P, cap = case["prefix"], case["cap"]
    s["q"] = normal(len(lens), H, hd, scale=1.5)
    s["prefix_k"], s["prefix_v"] = normal(KH, P, hd), normal(KH, P, hd, scale=0.7)
    s["k"], s["v"] = normal(len(lens), KH, cap, hd), normal(len(lens), KH, cap, hd, scale=0.7)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["max_len"] = max(lens)
    s["weights"] = torch.rand(len(lens), KH, cap, generator=g, device=dev) if case["weights"] else None
    return s


def run(state):
    s = state
    if own:
        from tinygiant_b200 import attention as A
        if s["op"] == "prompt":
            return A.attention_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_k=s["max_k"], window=s["window"],
                                      sinks=s["sinks"])
        if s["op"] == "shared":
            out = A.attention_shared(s["q"], s["prefix_k"], s["prefix_v"], s["k"], s["v"], s["lens"], max_len=s["max_len"],
                                     window=s["window"], sinks=s["sinks"], weights=s["weights"])
            return out if s["weights"] is None else (out, s["weights"])
        return A.cache_evict(s["k"], s["v"], s["weights"], s["lens"], s["keep"], s["recent"])
    if s["op"] == "prompt":
        return _plain_prompt(s)
    if s["op"] == "shared":
        return _plain_shared(s)
    return _plain_evict(s)


def _softmax(scores, sinks):
    """exp(scores - max) over the last axis in place, and 1 / (its sum and the sinks'); rows without a key give zeros."""
    top = scores.amax(-1, keepdim=True) if scores.shape[-1] else scores.new_full((*scores.shape[:-1], 1), -math.inf)
    if sinks is not None:
        top = torch.maximum(top, sinks)
    top = torch.where(top == -math.inf, 0.0, top)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    return scores, torch.where(total == 0, 0.0, 1 / total)


def _plain_prompt(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    (tq, H, hd), (tk, KH, _) = q.shape, k.shape
    dev = q.device
    iq, ik = torch.arange(tq, device=dev, dtype=torch.int32), torch.arange(tk, device=dev, dtype=torch.int32)
    sq = torch.searchsorted(s["cu_q"], iq, right=True) - 1       # the sequence of each row and key
    sk = torch.searchsorted(s["cu_k"], ik, right=True) - 1
    at = iq - s["cu_q"][sq + 1] + s["cu_k"][sq + 1]              # each row's own key, among the packed ones
    gone = (sq[:, None] != sk) | (ik > at[:, None])
    if s["window"]:
        gone |= ik <= at[:, None] - s["window"]
    qs = (q * (1 / math.sqrt(hd))).view(tq, KH, H // KH, hd).permute(1, 2, 0, 3).reshape(KH, H // KH * tq, hd)
    scores = torch.matmul(qs, k.permute(1, 2, 0)).view(KH, H // KH, tq, tk)
    scores.masked_fill_(gone, -math.inf)
    p, inv = _softmax(scores, None if s["sinks"] is None else s["sinks"].view(KH, H // KH, 1, 1))
    o = torch.matmul(p.view(KH, H // KH * tq, tk), v.permute(1, 0, 2)).view(KH, H // KH, tq, hd) * inv
    return o.permute(2, 0, 1, 3).reshape(tq, H, hd).to(s["q"].dtype)


def _plain_shared(s):
    q, pk, pv = s["q"].float(), s["prefix_k"].float(), s["prefix_v"].float()
    (B, H, hd), (KH, P, _), cap = q.shape, pk.shape, s["k"].shape[2]
    G, dev = H // KH, q.device
    j = torch.arange(P + cap, device=dev, dtype=torch.int32)
    end = P + s["lens"][:, None]
    gone = (j >= end)                                            # [B, P + cap]
    if s["window"]:
        gone |= j < end - s["window"]
    there = ~gone[:, None, P:, None]
    k, v = torch.where(there, s["k"].float(), 0.0), torch.where(there, s["v"].float(), 0.0)
    qs = (q * (1 / math.sqrt(hd))).view(B, KH, G, hd)
    pre = torch.matmul(qs.transpose(0, 1).reshape(KH, B * G, hd), pk.transpose(1, 2)).view(KH, B, G, P).transpose(0, 1)
    scores = torch.cat([pre, torch.matmul(qs, k.transpose(2, 3))], -1)
    scores.masked_fill_(gone[:, None, None], -math.inf)
    p, inv = _softmax(scores, None if s["sinks"] is None else s["sinks"].view(KH, G, 1))
    o = torch.matmul(p[..., :P].transpose(0, 1).reshape(KH, B * G, P), pv).view(KH, B, G, hd).transpose(0, 1)
    o = ((o + torch.matmul(p[..., P:], v)) * inv).reshape(B, H, hd).to(s["q"].dtype)
    if s["weights"] is None:
        return o
    s["weights"] += (p[..., P:] * inv).sum(2)
    return o, s["weights"]


def _plain_evict(s):
    k, v, w, keep = s["k"], s["v"], s["weights"], s["keep"]
    B, KH, cap, hd = k.shape
    j = torch.arange(cap, device=k.device)
    n = s["lens"][:, None, None].long()
    m = n.clamp(max=keep)                                        # positions that stay
    key = torch.where(j >= n - m.clamp(max=s["recent"]), math.inf, w)
    key = torch.where(j >= n, -math.inf, key)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    slot = torch.arange(keep, device=k.device).expand(B, KH, keep)
    idx = torch.sort(torch.where(slot < m, order, cap), dim=-1).values
    here = idx < cap
    at = torch.where(here, idx, 0)
    take = lambda x: torch.where(here[..., None], torch.gather(x, 2, at[..., None].expand(B, KH, keep, hd)), 0)  # noqa: E731
    return (take(k), take(v), torch.where(here, torch.gather(w, 2, at), 0.0), m.view(B).int(),
            torch.where(here, idx, -1).int())


def exact(case, seed):
    """From the definitions, sequence by sequence and head by head, in 64 bits."""
    s = prepare(case, seed)
    lens = _ints(case["lens"])
    if s["op"] == "evict":
        B, KH, cap, hd = s["k"].shape
        keep, w = s["keep"], s["weights"].double().cpu().numpy()
        import numpy as np
        idx = np.full((B, KH, keep), -1, np.int64)
        for b, n in enumerate(lens):
            m = min(n, keep)
            r = min(s["recent"], m)
            for h in range(KH):
                heavy = np.lexsort((np.arange(n - r), -w[b, h, :n - r]))[:m - r]
                idx[b, h, :m] = np.concatenate([np.sort(heavy), np.arange(n - r, n)])
        at = torch.from_numpy(idx).to(s["k"].device)
        b_, h_ = torch.arange(B, device=at.device)[:, None, None], torch.arange(KH, device=at.device)[None, :, None]
        none = at < 0
        pick = lambda x: x[b_, h_, at.clamp(min=0)].double()      # noqa: E731
        return (pick(s["k"]).masked_fill(none[..., None], 0), pick(s["v"]).masked_fill(none[..., None], 0),
                pick(s["weights"]).masked_fill(none, 0), torch.tensor([min(n, keep) for n in lens], dtype=torch.int32),
                at.int())
    H, KH, hd, window = case["heads"], case["kv_heads"], case["head_dim"], case["window"]

    def attend(q, k, v, first, head):
        """Rows q at positions first, first + 1, ... over keys at 0, 1, ...: the outputs and the softmax weights."""
        x = q.double() @ k.double().T / math.sqrt(hd)
        i, j = torch.arange(len(q), device=x.device)[:, None] + first, torch.arange(len(k), device=x.device)
        ok = (j <= i) & ((j > i - window) if window else True)
        x = torch.where(ok, x, -math.inf)
        if s["sinks"] is not None:
            x = torch.cat([x, s["sinks"][head].double().expand(len(q), 1)], 1)
        p = torch.nan_to_num(torch.softmax(x, 1), nan=0.0)[:, :len(k)]
        return p @ v.double(), p

    out = torch.zeros(*s["q"].shape, dtype=torch.float64, device=s["q"].device)
    if s["op"] == "prompt":
        cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
        for b in range(len(lens)):
            q, k, v = s["q"][cq[b]:cq[b + 1]], s["k"][ck[b]:ck[b + 1]], s["v"][ck[b]:ck[b + 1]]
            if len(q) == 0:
                continue
            for h in range(H):
                out[cq[b]:cq[b + 1], h] = attend(q[:, h], k[:, h * KH // H], v[:, h * KH // H], len(k) - len(q), h)[0]
        return out
    weights = None if s["weights"] is None else s["weights"].double()
    P = s["prefix_k"].shape[1]
    for b, n in enumerate(lens):
        for kh in range(KH):
            k = torch.cat([s["prefix_k"][kh], s["k"][b, kh, :n]])
            v = torch.cat([s["prefix_v"][kh], s["v"][b, kh, :n]])
            for h in range(kh * H // KH, (kh + 1) * H // KH):
                o, p = attend(s["q"][b, h][None], k, v, P + n - 1, h)
                out[b, h] = o[0]
                if weights is not None:
                    weights[b, kh, :n] += p[0, P:]
    return out if weights is None else (out, weights)
