"""A batch of requests served from a paged 8-bit cache through one decoder layer on the GPU.

    python examples/serve_paged.py [--batch 8] [--chunk 256] [--steps 48] [--page 64] [--drafts 3] [--window 0] [--bits 8]

The operators of tinygiant_b200.paged together with a resident mixture-of-
experts layer, as a server would call them.  Prompts arrive in chunks: each
chunk's queries and keys are normed and rotated (frequencies scaled for a
context eight times as long) as cache_append writes them to pages from a free
list, cache_gather reads the sequences' keys back, and attention_prompt attends
to them.  Then every step checks `drafts` drafted tokens beside the next one:
cache_append, attention_paged, and as many positions dropped as were wrong (here:
a number drawn beforehand).  Pages behind a window go back to the free list.
Weights are random.
"""
import argparse
import importlib.util
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))


def _serve_batch():
    spec = importlib.util.spec_from_file_location("serve_batch", ROOT / "examples" / "serve_batch.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


class Pages:
    """The pools, each sequence's table, and which pages are free."""

    def __init__(self, n_pages, batch, columns, kv_heads, page, head_dim, bits):
        import torch
        kind = torch.float8_e4m3fn if bits == 8 else torch.bfloat16
        self.k, self.v = (torch.zeros(n_pages, kv_heads, page, head_dim, dtype=kind, device="cuda") for _ in range(2))
        self.ks, self.vs = (torch.zeros(n_pages, kv_heads, page // 16, device="cuda") if bits == 8 else None for _ in range(2))
        self.page, self.free = page, list(range(n_pages))
        self.rows = [[-1] * columns for _ in range(batch)]
        self.tables = torch.full((batch, columns), -1, dtype=torch.int32, device="cuda")

    @property
    def scales(self):
        return {"k_scales": self.ks, "v_scales": self.vs}

    def cover(self, lens, window=0):
        """Pages for positions up to lens; those that no later token of a window will see are free again."""
        import torch
        changed = False
        for row, n in zip(self.rows, lens):
            for i in range(-(-n // self.page)):
                gone = window > 0 and (i + 1) * self.page <= n - window
                if gone and row[i] >= 0:
                    self.free.append(row[i])
                    row[i], changed = -2, True                   # never again
                elif not gone and row[i] == -1:
                    row[i], changed = self.free.pop(), True
        if changed:
            self.tables.copy_(torch.tensor(self.rows, dtype=torch.int32))


def serve(layer, prompts_x, chunk, steps, page, drafts, window, bits):
    """prompts_x: a list of [n, D].  Returns the last outputs, lengths, and what the last attention saw (for checks)."""
    import torch

    from tinygiant_b200 import attention as A
    from tinygiant_b200 import paged as P
    sb = _serve_batch()
    H, KH, HD, dev, B = sb.H, sb.KH, sb.HD, prompts_x[0].device, len(prompts_x)
    freqs, amplitude = P.rotary_frequencies(HD, 1e6, scaling="yarn", factor=8, original_len=4096, device=dev)
    ones = torch.ones(HD, device=dev)
    rope = {"freqs": freqs, "amplitude": amplitude, "q_norm": ones, "k_norm": ones}
    ends = lambda ns: torch.tensor([sum(ns[:i]) for i in range(len(ns) + 1)], dtype=torch.int32, device=dev)  # noqa: E731
    most = max(len(x) for x in prompts_x) + steps * (drafts + 1)
    columns = -(-most // page)
    cache = Pages(B * columns, B, columns, KH, page, HD, bits)
    lens = [0] * B
    # prompts, a chunk of each at a time
    last = [None] * B
    for at in range(0, max(len(x) for x in prompts_x), chunk):
        parts = [x[at:at + chunk] for x in prompts_x]
        new = [len(x) for x in parts]
        lens = [a + b for a, b in zip(lens, new)]
        cache.cover(lens)
        x = torch.cat(parts)
        q, k, v = layer.qkv(x)
        cu, n = ends(lens), torch.tensor(lens, dtype=torch.int32, device=dev)
        q = P.cache_append(k, v, cache.k, cache.v, cache.tables, n, ends(new), **cache.scales, **rope, q=q)
        keys, vals = P.cache_gather(cache.k, cache.v, cache.tables, cu, sum(lens), **cache.scales)
        x = layer.after(x, A.attention_prompt(q, keys, vals, ends(new), cu, max_k=max(lens), window=window))
        for b, y in enumerate(x.split(new)):
            last[b] = y[-1] if len(y) else last[b]
    tok = torch.stack(last)
    # decoding: the next token and its drafts
    right = torch.randint(0, drafts + 1, (steps, B), generator=torch.Generator().manual_seed(3)).tolist()
    n1, seen = drafts + 1, None
    for step in range(steps):
        lens = [n + n1 for n in lens]
        cache.cover(lens)
        x = (tok[:, None] * (1 + 0.01 * torch.arange(n1, device=dev)[:, None])).reshape(B * n1, -1)   # stand-ins for drafted tokens
        q, k, v = layer.qkv(x)
        n = torch.tensor(lens, dtype=torch.int32, device=dev)
        q = P.cache_append(k, v, cache.k, cache.v, cache.tables, n, **cache.scales, **rope, q=q).view(B, n1, H, HD)
        attn = P.attention_paged(q, cache.k, cache.v, cache.tables, n, **cache.scales, max_len=max(lens), window=window)
        seen = (q, cache, list(lens), attn, window)
        if step + 1 < steps:
            x = layer.after(x, attn).view(B, n1, -1)
            keep = right[step]
            lens = [a - drafts + r for a, r in zip(lens, keep)]
            tok = torch.stack([x[b, r] for b, r in enumerate(keep)])
            tok = tok * (tok.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
            cache.cover(lens, window)
    return tok, lens, seen


def check(seen):
    """The largest error of the last step's attention against its definition in fp32 over what the cache holds, over the largest output."""
    import torch

    from tinygiant_b200 import paged as P
    q, cache, lens, attn, window = seen
    B, n, H, HD = q.shape
    cu = torch.tensor([sum(lens[:i]) for i in range(B + 1)], dtype=torch.int32, device=q.device)
    keys, vals = (t.float() for t in P.cache_gather(cache.k, cache.v, cache.tables, cu, sum(lens), **cache.scales))
    worst = top = 0.0
    for b, m in enumerate(lens):
        k, v = keys[cu[b]:cu[b + 1]], vals[cu[b]:cu[b + 1]]
        j, e = torch.arange(m, device=q.device), torch.arange(m - n, m, device=q.device)[:, None]
        gone = (j > e) | ((j <= e - window) if window else False)
        x = torch.einsum("nkgd,jkd->kgnj", q[b].float().view(n, k.shape[1], -1, HD), k) * HD ** -0.5
        want = torch.einsum("kgnj,jkd->nkgd", torch.softmax(x.masked_fill(gone, float("-inf")), -1), v).reshape(n, H, HD)
        worst, top = max(worst, float((attn[b].float() - want).abs().max())), max(top, float(want.abs().max()))
    return worst / top


def main(argv=None):
    import torch
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("batch", 8), ("chunk", 256), ("steps", 48), ("page", 64), ("drafts", 3), ("window", 0), ("bits", 8)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args(argv)
    # a stream of its own: torch's default one is no stream that the layer could share
    with torch.cuda.stream(torch.cuda.Stream()):
        layer = _serve_batch().Layer(max_tokens=64)
        g = torch.Generator(device="cuda").manual_seed(1)
        prompts = [torch.randn(1 + (337 * b + 500) % 900, layer.D, generator=g, device="cuda") for b in range(a.batch)]
        args = (a.chunk, a.steps, a.page, a.drafts, a.window, a.bits)
        serve(layer, prompts, a.chunk, 2, *args[2:])
        torch.cuda.synchronize()
        t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        t0.record()
        tok, lens, seen = serve(layer, prompts, *args)
        t1.record()
        torch.cuda.synchronize()
        err, finite = check(seen), bool(torch.isfinite(tok).all())
        layer.close()
    cache = seen[1]
    print(f"{a.batch} requests of {min(map(len, prompts))} to {max(map(len, prompts))} tokens and {a.steps} steps of {a.drafts + 1} through one layer "
          f"in {t0.elapsed_time(t1):.2f} ms; {cache.k.shape[0] - len(cache.free)} of {cache.k.shape[0]} pages in use; last attention off by "
          f"{err:.1e} of its largest value")
    if not (err < 2e-2 and finite):
        raise SystemExit("the last attention does not match its definition")
    return err


if __name__ == "__main__":
    main()
