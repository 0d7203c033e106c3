"""A batch that shares a system prompt, decoded through one decoder layer on the GPU.

    python examples/serve_batch.py [--batch 8] [--prefix 512] [--steps 64] [--cap 160] [--keep 96]

The attention operators of tinygiant_b200.attention together with a resident
mixture-of-experts layer, as a server would call them: the system prompt and
the users' prompts go through attention_prompt, every new token through
attention_shared (which reads the system prompt's keys once for the batch and
gathers the weights of the others), caches that are full are cut down by
cache_evict, and the layer's experts follow each attention.  Weights are
random; RoPE and the norms of queries and keys are left out.
"""
import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

H, KH, HD = 32, 4, 128


class Layer:
    """Projections as bf16 matrices, the experts as a ResidentLayer."""

    def __init__(self, seed=0, n_experts=16, max_tokens=8):
        import torch

        import tinygiant_b200 as tg
        from tinygiant_b200 import synth
        from tinygiant_b200.layer import ResidentLayer
        self.lib = tg.load()
        self.moe = ResidentLayer(synth.qwen_layer(seed=seed, n_experts=n_experts, top_k=8), max_tokens=max_tokens)
        self.D = self.moe.D
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: (torch.randn(*s, generator=g, device="cuda") * s[0] ** -0.5).bfloat16()  # noqa: E731
        self.wqkv, self.wo = rand(self.D, (H + 2 * KH) * HD), rand(H * HD, self.D)
        self.lib.tg_cuda_set_stream(torch.cuda.current_stream().cuda_stream)   # one stream for both

    def qkv(self, x):
        """x [T, D] fp32: views of one product, q [T, H, hd], k and v [T, KH, hd]."""
        y = (x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()).bfloat16() @ self.wqkv
        y = y.view(len(x), H + 2 * KH, HD)
        return y[:, :H], y[:, H:H + KH], y[:, H + KH:]

    def after(self, x, attn):
        """x + the output projection, then the experts of every row added."""
        import torch

        import tinygiant_b200 as tg
        x = x + (attn.reshape(len(x), H * HD) @ self.wo).float()
        for t in range(0, len(x), self.moe.max_tokens):
            rows = x[t:t + self.moe.max_tokens].contiguous()
            out = torch.empty_like(rows)
            self.lib.tg_layer_forward_dev(self.moe.h, rows.data_ptr(), None, None, out.data_ptr(), len(rows), 1, None)
            tg.check(self.lib)
            x[t:t + self.moe.max_tokens] += out
        return x

    def close(self):
        self.lib.tg_cuda_synchronize()
        self.lib.tg_cuda_set_stream(None)
        self.moe.close()


def serve(layer, prefix_x, prompts_x, steps, cap, keep, recent):
    """prefix_x [P, D]; prompts_x: a list of [n, D], n <= cap; a decoded token's
    output is the next one's input.  Returns the last outputs, the caches' lengths
    and what each step's attention saw (for checks)."""
    import torch

    from tinygiant_b200 import attention as A
    dev, B, P = prefix_x.device, len(prompts_x), len(prefix_x)
    ends = lambda ns: torch.tensor([sum(ns[:i]) for i in range(len(ns) + 1)], dtype=torch.int32, device=dev)  # noqa: E731
    # the system prompt, once
    q, pk, pv = layer.qkv(prefix_x)
    layer.after(prefix_x, A.attention_prompt(q, pk, pv, ends([P]), max_k=P))
    # the users' prompts in one pass, each behind the system prompt's keys
    lens = [len(x) for x in prompts_x]
    x = torch.cat(prompts_x)
    q, k, v = layer.qkv(x)
    ks, vs = k.split(lens), v.split(lens)
    keys = torch.cat([t for own in ks for t in (pk, own)])
    vals = torch.cat([t for own in vs for t in (pv, own)])
    x = layer.after(x, A.attention_prompt(q, keys, vals, ends(lens), ends([P + n for n in lens]), max_k=P + max(lens)))
    # decoding: the prompts' keys into caches, the system prompt's as they are
    kc, vc = (torch.zeros(B, KH, cap, HD, dtype=torch.bfloat16, device=dev) for _ in range(2))
    for b, n in enumerate(lens):
        kc[b, :, :n], vc[b, :, :n] = ks[b].transpose(0, 1), vs[b].transpose(0, 1)
    weights = torch.zeros(B, KH, cap, device=dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    tok = torch.stack([t[-1] for t in x.split(lens)])
    pk, pv = pk.transpose(0, 1), pv.transpose(0, 1)              # [KH, P, hd] views
    rows, longest, seen = torch.arange(B, device=dev), max(lens), None
    for _ in range(steps):
        if longest == cap:                                       # full: keep the heaviest and the newest
            k2, v2, w2, n, _ = A.cache_evict(kc, vc, weights, n, keep, recent)
            kc[:, :, :keep], vc[:, :, :keep], weights[:, :, :keep] = k2, v2, w2
            weights[:, :, keep:] = 0
            longest = keep
        q, k, v = layer.qkv(tok)
        kc[rows, :, n.long()], vc[rows, :, n.long()] = k, v
        n, longest = n + 1, longest + 1
        attn = A.attention_shared(q, pk, pv, kc, vc, n, max_len=longest, weights=weights)
        seen = (q, pk, pv, kc, vc, n, attn)
        tok = layer.after(tok, attn)
        tok = tok * (tok.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    return tok, n, seen


def check(seen):
    """The largest error of the last step's attention against its definition in fp32, over the largest output."""
    import torch
    q, pk, pv, kc, vc, n, attn = seen
    B, G = len(q), H // KH
    k = torch.cat([pk.expand(B, *pk.shape), kc], 2).float()
    v = torch.cat([pv.expand(B, *pv.shape), vc], 2).float()
    x = torch.einsum("bkgd,bkjd->bkgj", q.float().view(B, KH, G, HD), k) * HD ** -0.5
    gone = torch.arange(k.shape[2], device=q.device) >= pk.shape[1] + n[:, None]
    want = torch.softmax(x.masked_fill(gone[:, None, None], float("-inf")), -1) @ v
    return float((attn.float() - want.view(B, H, HD)).abs().max() / want.abs().max())


def main(argv=None):
    import torch
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("batch", 8), ("prefix", 512), ("steps", 64), ("cap", 160), ("keep", 96), ("recent", 32)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args(argv)
    layer = Layer()
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda n: torch.randn(n, layer.D, generator=g, device="cuda")  # noqa: E731
    prompts = [rand(1 + (37 * b + 90) % min(120, a.cap)) for b in range(a.batch)]
    prefix = rand(a.prefix)
    serve(layer, prefix.clone(), prompts, 2, a.cap, a.keep, a.recent)
    torch.cuda.synchronize()
    t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    t0.record()
    tok, n, seen = serve(layer, prefix.clone(), prompts, a.steps, a.cap, a.keep, a.recent)
    t1.record()
    torch.cuda.synchronize()
    err = check(seen)
    layer.close()
    print(f"{a.batch} sequences on a prefix of {a.prefix}: prompts and {a.steps} tokens each through one layer in "
          f"{t0.elapsed_time(t1):.2f} ms; {n.tolist()} own positions kept; last attention off by {err:.1e} of its largest value")
    if not (err < 2e-2 and bool(torch.isfinite(tok).all())):
        raise SystemExit("the last attention does not match its definition")
    return err


if __name__ == "__main__":
    main()
